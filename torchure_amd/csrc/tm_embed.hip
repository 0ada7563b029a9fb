// tm_embed.hip -- gfx950 kernels of the token embedding:
//   lookup      y_i = scale w[id_i]
//   gradient    dw[v] = scale * (sum over i with id_i = v of dy_i), to a whole table or added to one that is there
//
// Both are bound by memory: the lookup by the rows read and written, the gradient by dy and, far more, by the table that it
// fills (8192 tokens of 151,936 ids x 1024 in fp32: 34 MB and 622). The gradient takes three launches and no atomics on values,
// so that its bits are the same every time:
//
//   1. Tokens by id. Workgroup b has the ids with id % B = b (so that a vocabulary's frequent, low ids spread over
//      all of them). It reads all ids twice, eight a lane on their way together (one after the other they took 49 latencies
//      each time of 50,001 tokens): first it counts, in LDS, its own ids and the tokens of the workgroups before it, which places its
//      part of the list; then those that match wait in a queue in their order. Of 64 neighbours in a queue a wave finds each one's
//      equals by ballots, and the 64s take their places from the ids' cursors one after the other (ranked by comparing
//      with all before, 50,001 tokens of which an eighth had one id took the workgroup that has it 104 us; so 37). An id that is out of
//      range or the padding's is on no list.
//   2. Sums. A wave takes 32 entries of the list and one panel of columns, adds rows in order, and writes a
//      sum out where the id changes: to the table if all of the id's entries are its own, else to a partial sum. The other workgroups of
//      the launch fill the rows of ids that do not occur with zeros, which is most of the bytes.
//   3. Ids with entries in several waves: their partial sums, in order.
//
// Measured: 8192 tokens of 151,936 ids x 1024 in fp32: lookup 19 us (its rows out of the caches, as after a gradient's zeros; 7.5 in
// them), the three launches 10, 118 (656 MB at 5.6 TB/s; stores of zeros alone reach 6.7) and 6. 50,001 of 4096 x 777 in bf16: 22; 37,
// 23 (too few bytes on their way: rows of 512 are read at 2.1 TB/s in as many tokens and at 4.2 in four times as many) and 14.

#include <hip/hip_runtime.h>

#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "torchure_amd.h"
#include "tm_act.h"
#include "tm_internal.h"
#include "tm_units.h"

namespace {

using tm_units::get;
using tm_units::put;
using tm_units::Raw;
using tm_units::read;
using tm_units::values;

template <typename... A>
int fail(int code, const char* fmt, A... args) {
  return tm_internal_fail(code, fmt, args...);
}

int launched(const char* what) {
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? TM_OK : fail(TM_ELAUNCH, "%s: launch failed: %s", what, hipGetErrorString(err));
}

constexpr int kWave = 64;

// ---------------------------------------------------------------- lookup

struct Lookup {
  void* y;
  const void* w;
  const void* ids;
  int64_t ldw, vocab, n;
  int ids64, cols, lanes;  // lanes to a row: a power of two, up to 256
  float scale;
};

__device__ __forceinline__ int64_t id_at(const void* ids, int ids64, int64_t i) {
  return ids64 ? static_cast<const int64_t*>(ids)[i] : static_cast<const int32_t*>(ids)[i];
}

// An id that names no row gives a row of NaN: the ids are on the device, where the host cannot refuse them.
template <bool kW32, bool kY32>
__global__ __launch_bounds__(256) void lookup_kernel(Lookup a) {
  constexpr int kU = kW32 || kY32 ? 4 : 8, kAhead = 4;
  const int l = threadIdx.x & (a.lanes - 1), per = 256 / a.lanes;
  const int64_t step = static_cast<int64_t>(gridDim.x) * per;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * per + threadIdx.x / a.lanes; i < a.n; i += step) {
    const int64_t id = id_at(a.ids, a.ids64, i);
    const bool there = static_cast<uint64_t>(id) < static_cast<uint64_t>(a.vocab);
    const float scale = there ? a.scale : __builtin_nanf("");
    const int64_t from = there ? id * a.ldw : 0;
    for (int c0 = kU * l; c0 < a.cols; c0 += kU * a.lanes * kAhead) {
      Raw<kW32, kU> row[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int c = c0 + k * kU * a.lanes;
        row[k] = read<kW32, kU>(a.w, from + c, there ? a.cols - c : 0);
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int c = c0 + k * kU * a.lanes;
        float v[kU];
        values(v, row[k]);
#pragma unroll
        for (int e = 0; e < kU; ++e) v[e] = there ? v[e] * scale : scale;
        put<kY32, kU, true>(a.y, i * a.cols + c, v, a.cols - c);
      }
    }
  }
}

// ---------------------------------------------------------------- 1. tokens by id

constexpr int kGroupThreads = 1024, kGroupWaves = kGroupThreads / kWave, kMostLocal = 8192;
constexpr int kIds = 8;                                // ids a lane has on their way
constexpr int kQueue = 2048;                             // entries that wait for their places
constexpr int kPartWaves = kQueue / (kIds * kWave);    // waves of a round that surely fit
constexpr int kParts = kGroupWaves / kPartWaves;
static_assert(kQueue % kGroupThreads == 0 && kGroupWaves % kPartWaves == 0 && kMostLocal <= 1 << 16, "whole parts, 16-bit ids");

struct Segment {
  int32_t start, count;
};

// The workspace: how many tokens are on the list, the list (positions, and their ids), and for each id its part of it.
struct Lists {
  int32_t* total;
  int32_t* order;
  int32_t* id;
  Segment* segments;  // of id v at (v % B) * locals + v / B
  int log2_b, locals;
};

__device__ __forceinline__ int64_t segment_at(const Lists& t, int32_t id) {
  return static_cast<int64_t>(id & ((1 << t.log2_b) - 1)) * t.locals + (id >> t.log2_b);
}

// The sums of the lanes before this one.
__device__ __forceinline__ int wave_before(int v) {
  int s = v;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int o = __shfl_up(s, d, kWave);
    if ((threadIdx.x & 63) >= d) s += o;
  }
  return s - v;
}

// ... of the workgroup's threads, and of all in `sum`. `room`: a word a wave; two barriers.
__device__ __forceinline__ int block_before(int v, int* room, int& sum) {
  const int wave = threadIdx.x >> 6, before = wave_before(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) room[wave] = before + v;
  __syncthreads();
  int base = 0;
  sum = 0;
#pragma unroll
  for (int i = 0; i < kGroupWaves; ++i) {
    const int s = room[i];
    if (i < wave) base += s;
    sum += s;
  }
  return base + before;
}

template <typename Id>
__global__ __launch_bounds__(kGroupThreads) void embed_group_kernel(const Id* __restrict__ ids, int32_t n, int64_t vocab,
                                                                    int64_t padding, Lists t) {
  __shared__ int cursor[kMostLocal];
  __shared__ int room[kGroupWaves];
  __shared__ int queue_pos[kQueue];
  __shared__ uint16_t queue_local[kQueue];
  constexpr int kRound = kGroupThreads * kIds;
  const int mask = (1 << t.log2_b) - 1, b = blockIdx.x, tid = threadIdx.x, wave = tid >> 6, l = tid & 63;
  for (int i = tid; i < t.locals; i += kGroupThreads) cursor[i] = 0;
  __syncthreads();
  // A round's ids, 512 neighbours a wave, all on their way together (past the last token its id again: no branch, which would
  // have each waited for by itself: 50,001 32-bit ids 55 us for 39); then f(k, id, whether it is on the list).
  auto load = [&](Id (&id)[kIds], int round) {
#pragma unroll
    for (int k = 0; k < kIds; ++k) id[k] = ids[min(round + (wave * kIds + k) * kWave + l, n - 1)];
  };
  auto each = [&](const Id (&id)[kIds], int round, auto&& f) {
#pragma unroll
    for (int k = 0; k < kIds; ++k) {
      const int i = round + (wave * kIds + k) * kWave + l;
      const int64_t v = id[k];
      f(k, static_cast<int>(v), i < n && static_cast<uint64_t>(v) < static_cast<uint64_t>(vocab) && v != padding);
    }
  };
  int before = 0;
  for (int round = 0; round < n; round += kRound) {
    Id id[kIds];
    load(id, round);
    each(id, round, [&](int, int v, bool wanted) {
      before += wanted && (v & mask) < b;
      if (wanted && (v & mask) == b) atomicAdd(&cursor[v >> t.log2_b], 1);
    });
  }
  int base = 0;
  block_before(before, room, base);  // (its barriers are behind the counts, too)
  // counts -> places: eight neighbours a thread
  constexpr int kEach = kMostLocal / kGroupThreads;
  int count[kEach], sum = 0, all = 0;
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int at = tid * kEach + k;
    count[k] = at < t.locals ? cursor[at] : 0;
    sum += count[k];
  }
  int place = base + block_before(sum, room, all);
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int at = tid * kEach + k;
    if (at < t.locals) {
      cursor[at] = place;
      t.segments[static_cast<int64_t>(b) * t.locals + at] = {place, count[k]};
    }
    place += count[k];
  }
  if (b == mask && tid == 0) *t.total = base + all;
  if (!all) return;  // (of the whole workgroup)
  __syncthreads();

  // Puts a queue's entries in their places. Of 64 neighbours in it a wave finds each one's equals before it; the 64s then take their
  // places from the cursors one after the other.
  int queued = 0;
  auto drain = [&] {
    constexpr int kMine = kQueue / kGroupThreads;
    int local[kMine], pos[kMine], rank[kMine], equal[kMine], dest[kMine];
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
      const int q = (k * kGroupWaves + wave) * kWave + l;
      const bool in = q < queued;
      local[k] = in ? queue_local[q] : -1;
      pos[k] = in ? queue_pos[q] : 0;
      rank[k] = equal[k] = dest[k] = 0;
      uint64_t left = __ballot(in);
      while (left) {  // of the wave's lanes those of one id at a time
        const int key = __builtin_amdgcn_readlane(local[k], __ffsll(static_cast<unsigned long long>(left)) - 1);
        const uint64_t same = __ballot(local[k] == key);
        if (local[k] == key) {
          rank[k] = __popcll(same & ((uint64_t(1) << l) - 1));
          equal[k] = __popcll(same);
        }
        left &= ~same;
      }
    }
    const int groups = (queued + kWave - 1) / kWave;
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
      const int end = min(groups, (k + 1) * kGroupWaves);
      for (int g = k * kGroupWaves; g < end; ++g) {
        if (g == k * kGroupWaves + wave && local[k] >= 0) {
          const int at = cursor[local[k]];
          dest[k] = at + rank[k];
          if (rank[k] == 0) cursor[local[k]] = at + equal[k];
        }
        __syncthreads();
      }
    }
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
      if (local[k] >= 0) {
        t.order[dest[k]] = pos[k];
        t.id[dest[k]] = (local[k] << t.log2_b) | b;
      }
    }
    queued = 0;
  };
  for (int round = 0; round < n; round += kRound) {
    Id id[kIds];
    load(id, round);
    int local[kIds], in_wave[kIds], mine = 0;
    each(id, round, [&](int k, int v, bool wanted) {
      local[k] = wanted && (v & mask) == b ? v >> t.log2_b : -1;
      const uint64_t ballot = __ballot(local[k] >= 0);
      in_wave[k] = mine + __popcll(ballot & ((uint64_t(1) << l) - 1));
      mine += __popcll(ballot);
    });
    if (l == 0) room[wave] = mine;
    __syncthreads();
    // the waves before this one, and those of each part: a part always fits an empty queue
    int ahead = 0, part[kParts] = {}, found = 0;
#pragma unroll
    for (int w = 0; w < kGroupWaves; ++w) {
      const int s = room[w];
      if (w < wave) ahead += s;
      part[w / kPartWaves] += s;
      found += s;
    }
    auto put_in = [&](int at) {
#pragma unroll
      for (int k = 0; k < kIds; ++k) {
        if (local[k] >= 0) {
          queue_pos[at + in_wave[k]] = round + (wave * kIds + k) * kWave + l;
          queue_local[at + in_wave[k]] = static_cast<uint16_t>(local[k]);
        }
      }
    };
    if (queued && queued + found > kQueue) drain();
    if (queued + found <= kQueue) {
      put_in(queued + ahead);
      queued += found;
      __syncthreads();
    } else {
#pragma unroll
      for (int p = 0; p < kParts; ++p) {
        if (wave / kPartWaves == p) put_in(ahead);
        ahead -= part[p];
        queued = part[p];
        __syncthreads();
        if (queued) drain();
      }
    }
  }
  if (queued) drain();
}

// ---------------------------------------------------------------- 2. sums, and rows that do not occur

constexpr int kEntries = 32;  // of the list to a wave

struct Sums {
  void* dw;
  const void* dy;
  float* partial;  // of each 32 entries two rows: the id that comes from the entries before, the one that goes on behind
  int64_t ldw, lddy, vocab;
  int cols, panels;
  int64_t sum_blocks;
  float scale;
  Lists t;
};

// dw's row at `at` = scale * sum, or that added to what is there.
template <bool kW32, int kU, bool kAdd>
__device__ __forceinline__ void finish(const Sums& a, int32_t id, int c, float (&sum)[kU]) {
  const int64_t at = id * a.ldw + c;
  float old[kU] = {};
  if constexpr (kAdd) get<kW32>(old, a.dw, at, a.cols - c);
#pragma unroll
  for (int i = 0; i < kU; ++i) sum[i] = kAdd ? fmaf(sum[i], a.scale, old[i]) : sum[i] * a.scale;
  put<kW32, kU, !kAdd>(a.dw, at, sum, a.cols - c);
}

template <int kU>
__device__ __forceinline__ void keep(const Sums& a, int64_t row, int c, const float (&sum)[kU]) {
#pragma unroll
  for (int h = 0; h < kU; h += 4) {
    float q[4] = {sum[h], sum[h + 1], sum[h + 2], sum[h + 3]};
    put<true, 4>(a.partial, row * a.cols + c + h, q, a.cols - c - h);
  }
}

template <bool kW32, bool kY32, bool kAdd>
__global__ __launch_bounds__(256) void embed_sum_kernel(Sums a) {
  constexpr int kU = kW32 || kY32 ? 4 : 8, kAhead = 8;
  const int l = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // Rows that do not occur: one to a wave, through the caches (8192 tokens of 151,936 x 1024 in bf16 61 us; past them and four rows to a wave
  // 83. A row of 1024 in fp32 to a workgroup, a store a thread, 8% slower.)
  if (blockIdx.x >= a.sum_blocks) {
    const int64_t blocks = gridDim.x - a.sum_blocks;
    const float none[kU] = {};
    for (int64_t v = (blockIdx.x - a.sum_blocks) * 4 + wave; v < a.vocab; v += blocks * 4) {
      if (a.t.segments[segment_at(a.t, static_cast<int32_t>(v))].count) continue;
      for (int c = kU * l; c < a.cols; c += kU * kWave) put<kW32, kU>(a.dw, v * a.ldw + c, none, a.cols - c);
    }
    return;
  }
  const int64_t task = static_cast<int64_t>(blockIdx.x) * 4 + wave, chunk = task / a.panels;
  const int64_t first = chunk * kEntries;
  const int total = *a.t.total;
  if (first >= total) return;
  const int n = min(kEntries, static_cast<int>(total - first)), c = kU * (static_cast<int>(task - chunk * a.panels) * kWave + l);
  // lane j: entry j
  const int mine = min(l, n - 1);
  const int32_t pos = a.t.order[first + mine], id = a.t.id[first + mine];
  const Segment s = a.t.segments[segment_at(a.t, id)];
  const bool last = l < n && first + l + 1 == s.start + s.count;  // the id's last entry
  const uint64_t ends = __ballot(last || l == n - 1);
  const bool from_before = __builtin_amdgcn_readfirstlane(s.start) < first;
  const bool goes_on = !((__ballot(last) >> (n - 1)) & 1);
  const int left = a.cols - c;
  float sum[kU] = {};
  bool whole = !from_before;
  for (int j0 = 0; j0 < n; j0 += kAhead) {
    Raw<kY32, kU> row[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int32_t p = __builtin_amdgcn_readlane(pos, j0 + k);  // (lanes past n hold the last entry's)
      row[k] = read<kY32, kU, true>(a.dy, static_cast<int64_t>(p) * a.lddy + c, j0 + k < n ? left : 0);
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int j = j0 + k;
      if (j < n) {
        float v[kU];
        values(v, row[k]);
#pragma unroll
        for (int i = 0; i < kU; ++i) sum[i] += v[i];
        if ((ends >> j) & 1) {
          const bool open = j == n - 1 && goes_on;
          if (whole && !open) finish<kW32, kU, kAdd>(a, __builtin_amdgcn_readlane(id, j), c, sum);
          else keep(a, 2 * chunk + (whole ? 1 : 0), c, sum);
          whole = true;
#pragma unroll
          for (int i = 0; i < kU; ++i) sum[i] = 0.0f;
        }
      }
    }
  }
}

// ---------------------------------------------------------------- 3. ids of several waves

// A workgroup to the entries (blockIdx.x) in which an id begins that goes on behind, and a panel of columns (blockIdx.y): each of
// its 4 waves adds a part of the id's partial sums, in order, and the first the waves'.
template <bool kW32, bool kAdd>
__global__ __launch_bounds__(256) void embed_join_kernel(Sums a) {
  __shared__ float part[3][4][kWave];
  const int64_t chunk = blockIdx.x, next = (chunk + 1) * kEntries;
  const int total = *a.t.total;
  if (next >= total) return;
  const int32_t id = a.t.id[next - 1];
  const Segment s = a.t.segments[segment_at(a.t, id)];
  if (s.start < chunk * kEntries || s.start + s.count <= next) return;  // began before, or ends here
  const int64_t behind = (s.start + s.count - 1) / kEntries - chunk;    // how many more entries' waves it is in
  const int l = threadIdx.x & 63, wave = threadIdx.x >> 6, c = 4 * (static_cast<int>(blockIdx.y) * kWave + l), left = a.cols - c;
  const int64_t each = (behind + 4) / 4, begin = wave * each, end = min(behind + 1, begin + each);
  float sum[4] = {};
  constexpr int kAhead = 16;
  for (int64_t i = begin; i < end; i += kAhead) {
    Raw<true, 4> row[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t m = i + k;
      row[k] = read<true, 4>(a.partial, (2 * (chunk + m) + (m == 0 ? 1 : 0)) * a.cols + c, m < end ? left : 0);
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      float v[4];
      values(v, row[k]);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += v[e];
    }
  }
  if (wave) {
#pragma unroll
    for (int e = 0; e < 4; ++e) part[wave - 1][e][l] = sum[e];
  }
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int w = 0; w < 3; ++w)
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] += part[w][e][l];
  finish<kW32, 4, kAdd>(a, id, c, sum);
}

// ---------------------------------------------------------------- sizes

constexpr int64_t kMostTokens = int64_t(1) << 30, kMostVocab = int64_t(1) << 30, kMostCols = int64_t(1) << 20;

// Workgroups of the first launch: 256, one to a CU, or as many as leave each 8192 ids.
int log2_groups(int64_t vocab) {
  int b = 8;
  while ((vocab + (int64_t(1) << b) - 1) >> b > kMostLocal) ++b;
  return b;
}
int64_t locals_of(int64_t vocab, int log2_b) { return (vocab + (int64_t(1) << log2_b) - 1) >> log2_b; }
int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }
int64_t chunks_of(int64_t tokens) { return (tokens + kEntries - 1) / kEntries; }

int check_sizes(const char* who, int64_t tokens, int64_t vocab, int64_t cols) {
  if (tokens < 0 || tokens > kMostTokens || vocab < 1 || vocab > kMostVocab || cols < 1 || cols > kMostCols)
    return fail(TM_EINVAL, "%s: %lld tokens of %lld ids x %lld columns: at most 2^30, 1 to 2^30 and 1 to 2^20", who,
                (long long)tokens, (long long)vocab, (long long)cols);
  return TM_OK;
}

bool odd(const void* p, int size) { return (reinterpret_cast<uintptr_t>(p) & (size - 1)) != 0; }

template <class F>
void with_flag(bool flag, F&& f) {
  if (flag) f(std::true_type{});
  else f(std::false_type{});
}

}  // namespace

extern "C" {

int tm_embed_lookup(void* d_y, int y_f32, const void* d_w, int w_f32, int64_t ldw, const void* d_ids, int ids64, int64_t tokens,
                    int64_t vocab, int64_t cols, float scale, void* stream) {
  const char* who = "tm_embed_lookup";
  if (int rc = check_sizes(who, tokens, vocab, cols)) return rc;
  if (tokens == 0) return TM_OK;
  if (!d_y || !d_w || !d_ids) return fail(TM_EINVAL, "%s: null pointer", who);
  if (ldw < cols && vocab > 1) return fail(TM_EINVAL, "%s: rows %lld elements apart", who, (long long)ldw);
  if (odd(d_y, y_f32 ? 4 : 2) || odd(d_w, w_f32 ? 4 : 2) || odd(d_ids, ids64 ? 8 : 4))
    return fail(TM_EINVAL, "%s: a pointer that is not aligned to its elements", who);
  Lookup a = {d_y, d_w, d_ids, ldw, vocab, tokens, ids64, static_cast<int>(cols), 8, scale};
  // up to four units a lane, at least 8 lanes: neighbours' bytes in one access of a wave
  const int64_t units = (cols + (w_f32 || y_f32 ? 4 : 8) - 1) / (w_f32 || y_f32 ? 4 : 8);
  while (a.lanes < 256 && a.lanes * 4 < units) a.lanes *= 2;
  const int64_t per = 256 / a.lanes, blocks = std::min((tokens + per - 1) / per, int64_t(1) << 23);
  with_flag(w_f32, [&](auto w32) {
    with_flag(y_f32, [&](auto y32) {
      hipLaunchKernelGGL((lookup_kernel<decltype(w32)::value, decltype(y32)::value>), dim3(static_cast<uint32_t>(blocks)),
                         dim3(256), 0, static_cast<hipStream_t>(stream), a);
    });
  });
  return launched(who);
}

size_t tm_embed_grad_workspace_bytes(int64_t tokens, int64_t vocab, int64_t cols) {
  if (tokens < 1 || tokens > kMostTokens || vocab < 1 || vocab > kMostVocab || cols < 1 || cols > kMostCols) return 0;
  const int log2_b = log2_groups(vocab);
  return static_cast<size_t>(16 + 2 * up(4 * tokens, 16) + up(8 * (locals_of(vocab, log2_b) << log2_b), 16) +
                             8 * chunks_of(tokens) * cols);
}

int tm_embed_grad(void* d_dw, int w_f32, int64_t ldw, const void* d_dy, int y_f32, int64_t lddy, const void* d_ids, int ids64,
                  int64_t tokens, int64_t vocab, int64_t cols, float scale, int64_t padding, int add, void* d_ws,
                  size_t ws_bytes, void* stream) {
  const char* who = "tm_embed_grad";
  if (int rc = check_sizes(who, tokens, vocab, cols)) return rc;
  if (tokens == 0) return fail(TM_EINVAL, "%s: no tokens", who);
  if (!d_dw || !d_dy || !d_ids) return fail(TM_EINVAL, "%s: null pointer", who);
  if ((ldw < cols && vocab > 1) || (lddy < cols && tokens > 1))
    return fail(TM_EINVAL, "%s: rows %lld and %lld elements apart", who, (long long)ldw, (long long)lddy);
  if (odd(d_dw, w_f32 ? 4 : 2) || odd(d_dy, y_f32 ? 4 : 2) || odd(d_ids, ids64 ? 8 : 4))
    return fail(TM_EINVAL, "%s: a pointer that is not aligned to its elements", who);
  const size_t need = tm_embed_grad_workspace_bytes(tokens, vocab, cols);
  if (!d_ws || ws_bytes < need || odd(d_ws, 16))
    return fail(TM_EINVAL, "%s: workspace of %zu bytes, %zu needed, aligned to 16", who, d_ws ? ws_bytes : size_t(0), need);
  const int log2_b = log2_groups(vocab);
  char* ws = static_cast<char*>(d_ws);
  Lists t;
  t.log2_b = log2_b;
  t.locals = static_cast<int>(locals_of(vocab, log2_b));
  t.total = reinterpret_cast<int32_t*>(ws);
  ws += 16;
  t.order = reinterpret_cast<int32_t*>(ws);
  ws += up(4 * tokens, 16);
  t.id = reinterpret_cast<int32_t*>(ws);
  ws += up(4 * tokens, 16);
  t.segments = reinterpret_cast<Segment*>(ws);
  ws += up(8 * (static_cast<int64_t>(t.locals) << log2_b), 16);
  const bool wide = w_f32 || y_f32;
  const int64_t units = (cols + (wide ? 4 : 8) - 1) / (wide ? 4 : 8), panels = (units + kWave - 1) / kWave;
  const int64_t chunks = chunks_of(tokens), sum_blocks = (chunks * panels + 3) / 4;
  const int64_t fill_blocks = add ? 0 : std::min<int64_t>((vocab + 3) / 4, 1 << 20);
  const int64_t join_panels = (cols + 4 * kWave - 1) / (4 * kWave);
  if (sum_blocks + fill_blocks >= int64_t(1) << 24 || (chunks - 1) * join_panels >= int64_t(1) << 24)  // of 256: less than 2^32 a launch
    return fail(TM_EINVAL, "%s: %lld tokens x %lld columns are too large for a launch", who, (long long)tokens, (long long)cols);
  const Sums a = {d_dw, d_dy, reinterpret_cast<float*>(ws), ldw, lddy, vocab, static_cast<int>(cols),
                  static_cast<int>(panels), sum_blocks, scale, t};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 groups(uint32_t(1) << log2_b);
  if (ids64) hipLaunchKernelGGL(embed_group_kernel<int64_t>, groups, dim3(kGroupThreads), 0, s,
                                static_cast<const int64_t*>(d_ids), static_cast<int32_t>(tokens), vocab, padding, t);
  else hipLaunchKernelGGL(embed_group_kernel<int32_t>, groups, dim3(kGroupThreads), 0, s, static_cast<const int32_t*>(d_ids),
                          static_cast<int32_t>(tokens), vocab, padding, t);
  if (int rc = launched("embed_group_kernel")) return rc;
  with_flag(w_f32, [&](auto w32) {
    with_flag(y_f32, [&](auto y32) {
      with_flag(add, [&](auto adds) {
        hipLaunchKernelGGL((embed_sum_kernel<decltype(w32)::value, decltype(y32)::value, decltype(adds)::value>),
                           dim3(static_cast<uint32_t>(sum_blocks + fill_blocks)), dim3(256), 0, s, a);
      });
    });
  });
  if (int rc = launched("embed_sum_kernel")) return rc;
  if (chunks < 2) return TM_OK;
  const dim3 joins(static_cast<uint32_t>(chunks - 1), static_cast<uint32_t>(join_panels));
  with_flag(w_f32, [&](auto w32) {
    with_flag(add, [&](auto adds) {
      hipLaunchKernelGGL((embed_join_kernel<decltype(w32)::value, decltype(adds)::value>), joins, dim3(256), 0, s, a);
    });
  });
  return launched("embed_join_kernel");
}

}  // extern "C"
