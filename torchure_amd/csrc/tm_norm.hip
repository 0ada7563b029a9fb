// tm_norm.hip -- gfx950 kernels of layer norm and RMS norm over a matrix's rows, forward and backward.
//
//   forward    xhat = (x - mean) rstd,  rstd = 1 / sqrt(mean((x - mean)^2) + eps),  y = xhat w + b   (RMS: mean = 0)
//   backward   g = dy w,  dx = rstd (g - mean(g xhat) xhat - mean(g)),  dw = sum over rows of dy xhat,  db = of dy
//              (RMS: without mean(g) and db)
//
// Both are bound by memory: x in, y out; x and dy in, dx out. A row stays in the registers of the lanes that it is dealt to, between
// its loads and its results, so the statistics take two passes over registers (the sum of squared distances from the mean, not of
// squares) and no second read. A row has 8 to 64 lanes of a wave, or a workgroup of 8 waves, by its length; lanes
// that share a row add by DPP moves and readlane, waves over LDS. A workgroup takes rows at the grid's stride, with the weight in
// registers. The weight's gradient is summed in registers over the rows that a wave takes, then over the workgroup's waves,
// and the workgroups' sums, in order, by a second launch: no atomics, the same bits every time.

#include <hip/hip_runtime.h>

#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "torchure_amd.h"
#include "tm_act.h"
#include "tm_internal.h"
#include "tm_units.h"

namespace {

using tm_act::bf16_lo;
using tm_act::pack_bf16;
using tm_units::get;
using tm_units::put;
using tm_units::Raw;
using tm_units::read;
using tm_units::values;

template <typename... A>
int fail(int code, const char* fmt, A... args) {
  return tm_internal_fail(code, fmt, args...);
}

constexpr int kWave = 64;
constexpr int kCus = 256;
constexpr float kMost = 0x1.fffffep127f;
// Results go past the caches: 8192 x 2560 forward 16.7 us for 20.9, fp32 8192 x 1024 backward 14.7 for 18.1; a product of 9728 columns
// behind the first takes the same time with it either way (338-341 us).
constexpr bool kStream = true;

// ---------------------------------------------------------------- sums over a row's lanes

template <int kCtrl>
__device__ __forceinline__ float moved(float v) {
  return __uint_as_float(static_cast<uint32_t>(
      __builtin_amdgcn_update_dpp(0, static_cast<int>(__float_as_uint(v)), kCtrl, 0xF, 0xF, true)));
}
__device__ __forceinline__ float lane(float v, int i) {
  return __uint_as_float(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(__float_as_uint(v)), i)));
}

// The sum over each group of kLanes neighbours, the same bits in each of them.
template <int kLanes>
__device__ __forceinline__ float group_sum(float v) {
  static_assert(kLanes == 8 || kLanes == 16 || kLanes == 32 || kLanes == 64, "");
  v += moved<0xB1>(v);   // lane ^ 1
  v += moved<0x4E>(v);   // lane ^ 2
  v += moved<0x141>(v);  // the other four of eight
  if constexpr (kLanes >= 16) v += moved<0x140>(v);  // the other eight of sixteen
  if constexpr (kLanes >= 32) {
    const float a = lane(v, 0) + lane(v, 16), b = lane(v, 32) + lane(v, 48);
    if constexpr (kLanes == 64) return a + b;
    else return (threadIdx.x & 32) ? b : a;
  }
  return v;
}

// kN sums over a row: its kLanes lanes, or the workgroup's. `room`: 2 x 16 floats of LDS used in turn: a wave writes one half
// again only after a barrier that every wave reaches when it has read it.
template <int kLanes>
struct RowSum {
  float* room;
  int turn = 0;
  template <int kN>
  __device__ __forceinline__ void operator()(float (&v)[kN]) {
#pragma unroll
    for (int n = 0; n < kN; ++n) v[n] = group_sum<kLanes < kWave ? kLanes : kWave>(v[n]);
    if constexpr (kLanes > kWave) {
      constexpr int kWaves = kLanes / kWave;
      static_assert(kN * kWaves <= 16, "");
      float* r = room + 16 * turn;
      turn ^= 1;
      if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (int n = 0; n < kN; ++n) r[n * kWaves + (threadIdx.x >> 6)] = v[n];
      }
      __syncthreads();
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        v[n] = r[n * kWaves];
#pragma unroll
        for (int i = 1; i < kWaves; ++i) v[n] += r[n * kWaves + i];
      }
    }
  }
  __device__ __forceinline__ float operator()(float v) {
    float one[1] = {v};
    (*this)(one);
    return one[0];
  }
};

// A kernel's shape: kLanes lanes to a row, kVec units of kU elements to a lane; workgroups of whole rows.
template <int kLanes_, int kVec_, int kU_>
struct Shape {
  static constexpr int kLanes = kLanes_, kVec = kVec_, kU = kU_;
  static constexpr int kEach = kVec * kU;  // elements of a lane
  static constexpr int kForwardThreads = kLanes <= kWave ? 256 : kLanes;
  static constexpr int kBackwardThreads = kLanes <= kWave ? 256 : kLanes;
};

struct Forward {
  void* y;
  float* rstd;
  float* mean;
  const void* x;
  const void* w;
  const void* b;
  int64_t ldx, rows;
  int cols;
  int w_f32, b_f32;
  float eps, inv_cols;
};

// A unit of a weight or bias of either type, or `otherwise`.
template <int kU>
__device__ __forceinline__ void param(float (&v)[kU], const void* p, int f32, int at, int cols, float otherwise) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < kU; ++i) v[i] = otherwise;
  } else if (f32) {
#pragma unroll
    for (int h = 0; h < kU; h += 4) {
      float q[4];
      get<true>(q, p, at + h, cols - at - h);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[h + i] = q[i];
    }
  } else {
    get<false>(v, p, at, cols - at);
  }
}

// A row's units as this lane reads them; `cols` is 0 for a row that is not there.
template <class S, bool kF32>
struct Row {
  Raw<kF32, S::kU> u[S::kVec];
  __device__ __forceinline__ void load(const void* base, int64_t at, int l, int cols) {
#pragma unroll
    for (int k = 0; k < S::kVec; ++k) {
      const int c = S::kU * (l + k * S::kLanes);
      u[k] = read<kF32, S::kU>(base, at + c, cols - c);
    }
  }
};

template <class S, bool kX32, bool kY32, bool kLayer>
__global__ __launch_bounds__(S::kForwardThreads) void norm_forward_kernel(Forward a) {
  constexpr int kRows = S::kForwardThreads / S::kLanes;  // of a workgroup at a time
  __shared__ float room[32];
  RowSum<S::kLanes> row_sum{room};
  const int l = threadIdx.x % S::kLanes, mine = threadIdx.x / S::kLanes;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  int64_t r0 = static_cast<int64_t>(blockIdx.x) * kRows;
  Row<S, kX32> next;
  next.load(a.x, (r0 + mine) * a.ldx, l, r0 + mine < a.rows ? a.cols : 0);
  float w[S::kVec][S::kU], b[S::kVec][S::kU];
#pragma unroll
  for (int k = 0; k < S::kVec; ++k) {
    const int c = S::kU * (l + k * S::kLanes);
    param(w[k], a.w, a.w_f32, c, a.cols, 1.0f);
    param(b[k], a.b, a.b_f32, c, a.cols, 0.0f);
  }
  for (; r0 < a.rows; r0 += step) {
    const int64_t r = r0 + mine;
    const int cols = r < a.rows ? a.cols : 0;
    float x[S::kVec][S::kU];
#pragma unroll
    for (int k = 0; k < S::kVec; ++k) values(x[k], next.u[k]);
    // the next row is on its way while this one is worked on
    if (r0 + step < a.rows) next.load(a.x, (r + step) * a.ldx, l, r + step < a.rows ? a.cols : 0);
    float mean = 0.0f;
    if constexpr (kLayer) {
      float s = 0.0f;
#pragma unroll
      for (int k = 0; k < S::kVec; ++k)
#pragma unroll
        for (int i = 0; i < S::kU; ++i) s += x[k][i];
      mean = row_sum(s) * a.inv_cols;
    }
    float q = 0.0f;
#pragma unroll
    for (int k = 0; k < S::kVec; ++k)
#pragma unroll
      for (int i = 0; i < S::kU; ++i) {
        x[k][i] -= mean;
        const float d = S::kU * (l + k * S::kLanes) + i < cols ? x[k][i] : 0.0f;
        q = fmaf(d, d, q);
      }
    const float rstd = 1.0f / sqrtf(fmaf(row_sum(q), a.inv_cols, a.eps));
    if (a.rstd && l == 0 && cols) {
      a.rstd[r] = rstd;
      if constexpr (kLayer) a.mean[r] = mean;
    }
#pragma unroll
    for (int k = 0; k < S::kVec; ++k) {
      const int c = S::kU * (l + k * S::kLanes);
      float y[S::kU];
#pragma unroll
      for (int i = 0; i < S::kU; ++i) y[i] = fmaf(x[k][i] * rstd, w[k][i], b[k][i]);
      put<kY32, S::kU, kStream>(a.y, r * a.cols + c, y, cols - c);
    }
  }
}

struct Backward {
  void* dx;          // or NULL
  float* dw;         // workgroups x cols, or NULL
  float* db;         // likewise
  const void* x;
  const void* dy;
  const void* w;
  const float* rstd;
  const float* mean;
  int64_t ldx, lddy, rows;
  int cols;
  int w_f32;
  float inv_cols;
};

// kParams: dw and db are wanted. A row's x and dy stay as they were read and are widened twice, for the sums and for dx, and the
// weight is in LDS: what a lane holds for long is the sums of dw and db (40 + 40 registers at 2560 columns).
template <class S, bool kX32, bool kY32, bool kLayer, bool kParams>
__global__ __launch_bounds__(S::kBackwardThreads) void norm_backward_kernel(Backward a) {
  constexpr int kRows = S::kBackwardThreads / S::kLanes, kWide = S::kLanes * S::kEach;
  // A wave's row has the next one on its way. In workgroups of 8 waves, one or two to a CU, that would fit their 256
  // registers and gains nothing (layer norm backward of 4096 x 9728 in bf16 58 us either way, in fp32 96 without and 100 with it,
  // RMS 8192 x 6144 63 and 66).
  constexpr bool kAhead = S::kLanes <= kWave;
  __shared__ float room[32];
  __shared__ float weight[kWide];
  __shared__ float part[kParams && kRows > 1 ? kRows : 1][kParams && kRows > 1 ? kWide : 1];
  RowSum<S::kLanes> row_sum{room};
  const int l = threadIdx.x % S::kLanes, mine = threadIdx.x / S::kLanes;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  int64_t r0 = static_cast<int64_t>(blockIdx.x) * kRows;
  Row<S, kX32> next_x;
  Row<S, kY32> next_dy;
  auto load = [&](int64_t r) {
    const int cols = r < a.rows ? a.cols : 0;
    next_x.load(a.x, r * a.ldx, l, a.x ? cols : 0);
    next_dy.load(a.dy, r * a.lddy, l, cols);
  };
  if constexpr (kAhead) load(r0 + mine);
  for (int c = S::kU * threadIdx.x; c < kWide; c += S::kU * S::kBackwardThreads) {
    float w[S::kU];
    param(w, a.w, a.w_f32, c, a.cols, 1.0f);
#pragma unroll
    for (int i = 0; i < S::kU; ++i) weight[c + i] = w[i];
  }
  __syncthreads();
  float dw[kParams ? S::kVec : 1][S::kU] = {}, db[kParams && kLayer ? S::kVec : 1][S::kU] = {};
  for (; r0 < a.rows; r0 += step) {
    const int64_t r = r0 + mine;
    const int cols = r < a.rows ? a.cols : 0;
    const bool there = cols && a.x;  // (x is left out where db alone is wanted)
    const float rstd = there ? a.rstd[r] : 0.0f, mean = kLayer && there ? a.mean[r] : 0.0f;
    // Where mean rstd passes fp32 (both finite), all of the row is its mean: a distance of even 2^-48 of it would make rstd less. Its
    // xhat is 0, but past its end, where x is read as 0, it is -inf, and times a g of 0 NaN.
    const bool far = kLayer && fabsf(mean * rstd) > kMost && fabsf(mean) <= kMost && rstd <= kMost;
    if constexpr (!kAhead) load(r);
    const Row<S, kX32> row_x = next_x;
    const Row<S, kY32> row_dy = next_dy;
    if constexpr (kAhead) {
      if (r0 + step < a.rows) load(r + step);
    }
    // v[0] = sum of g xhat, v[1] = sum of g
    float v[kLayer ? 2 : 1] = {};
#pragma unroll
    for (int k = 0; k < S::kVec; ++k) {
      const float* w = weight + S::kU * (l + k * S::kLanes);
      float x[S::kU], dy[S::kU];
      values(x, row_x.u[k]);
      values(dy, row_dy.u[k]);
#pragma unroll
      for (int i = 0; i < S::kU; ++i) {
        const float xhat = (x[i] - mean) * rstd, g = dy[i] * w[i];
        if constexpr (kParams) {
          dw[k][i] = fmaf(dy[i], xhat, dw[k][i]);
          if constexpr (kLayer) db[k][i] += dy[i];
        }
        v[0] = fmaf(g, xhat, v[0]);
        if constexpr (kLayer) v[1] += g;
      }
    }
    row_sum(v);
    const float along = far ? 0.0f : v[0] * a.inv_cols, mid = kLayer ? v[kLayer ? 1 : 0] * a.inv_cols : 0.0f;
    if (a.dx) {
#pragma unroll
      for (int k = 0; k < S::kVec; ++k) {
        const int c = S::kU * (l + k * S::kLanes);
        const float* w = weight + c;
        float x[S::kU], dy[S::kU], dx[S::kU];
        values(x, row_x.u[k]);
        values(dy, row_dy.u[k]);
#pragma unroll
        for (int i = 0; i < S::kU; ++i) dx[i] = (fmaf(dy[i], w[i], -mid) - (x[i] - mean) * rstd * along) * rstd;
        put<kX32, S::kU, kStream>(a.dx, r * a.cols + c, dx, cols - c);
      }
    }
  }
  if constexpr (kParams) {
    // over the workgroup's rows, in order
#pragma unroll
    for (int which = 0; which < (kLayer ? 2 : 1); ++which) {
      float* out = which ? a.db : a.dw;
      if (!out) continue;
      out += static_cast<int64_t>(blockIdx.x) * a.cols;
      if (kRows > 1 && which) __syncthreads();
#pragma unroll
      for (int k = 0; k < S::kVec; ++k) {
        const int c = S::kU * (l + k * S::kLanes);
        const float(&sums)[S::kU] = which ? db[kLayer ? k : 0] : dw[k];
        if constexpr (kRows == 1) {
          put<true, 4>(out, c, reinterpret_cast<const float(&)[4]>(sums[0]), a.cols - c);
          if constexpr (S::kU == 8) put<true, 4>(out, c + 4, reinterpret_cast<const float(&)[4]>(sums[4]), a.cols - c - 4);
        } else {
#pragma unroll
          for (int i = 0; i < S::kU; ++i) part[mine][c + i] = sums[i];
        }
      }
      if constexpr (kRows > 1) {
        __syncthreads();
        for (int c = threadIdx.x; c < kWide; c += S::kBackwardThreads) {
          float s = part[0][c];
#pragma unroll
          for (int j = 1; j < kRows; ++j) s += part[j][c];
          if (c < a.cols) out[c] = s;
        }
      }
    }
  }
}

// out (blockIdx.y: dw, db) = the sums over the workgroups' rows of `parts`, each of 16 waves a sixteenth of them in order.
struct Join {
  const float* parts[2];
  void* out[2];
  int f32[2];
  int n, cols;
};
__global__ __launch_bounds__(1024) void norm_join_kernel(Join a) {
  __shared__ float part[16][kWave];
  const int wave = threadIdx.x >> 6, l = threadIdx.x & 63, c = blockIdx.x * kWave + l;
  const float* p = a.parts[blockIdx.y];
  void* out = a.out[blockIdx.y];
  if (!out) return;
  const int each = (a.n + 15) / 16, first = wave * each, last = min(a.n, first + each);
  float s = 0.0f;
  if (c < a.cols) {
    constexpr int kAhead = 16;
    for (int i = first; i < last; i += kAhead) {
      float v[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) v[j] = i + j < last ? p[static_cast<int64_t>(i + j) * a.cols + c] : 0.0f;
#pragma unroll
      for (int j = 0; j < kAhead; ++j) s += v[j];
    }
  }
  part[wave][l] = s;
  __syncthreads();
  if (wave || c >= a.cols) return;
  for (int i = 1; i < 16; ++i) s += part[i][l];
  if (a.f32[blockIdx.y]) static_cast<float*>(out)[c] = s;
  else static_cast<uint16_t*>(out)[c] = static_cast<uint16_t>(pack_bf16(s, s));
}

// ---------------------------------------------------------------- which shape, how many workgroups

constexpr int kMaxCols = 16384;

// f(Shape) for rows of `cols` columns: the fewest lanes and units that hold them. A row is one wave's up to 40 or 48 elements a
// lane, past that a workgroup's of eight waves. The backward pass holds a lane's elements up to six times: with layer norm's dw and db
// 166 to 256 registers at 20 to 32 of them, at 40 and 48 all 256 and 24 to 72 values in accumulation registers, one wave to a SIMD.
template <int kU, class F>
int with_shape(int cols, F&& f) {
  const int units = (cols + kU - 1) / kU;
  if (units <= 8) return f(Shape<8, 1, kU>{});
  if (units <= 16) return f(Shape<16, 1, kU>{});
  if (units <= 32) return f(Shape<32, 1, kU>{});
  switch ((units + 63) / 64) {
    case 1: return f(Shape<64, 1, kU>{});
    case 2: return f(Shape<64, 2, kU>{});
    case 3: return f(Shape<64, 3, kU>{});
    case 4: return f(Shape<64, 4, kU>{});
    case 5: return f(Shape<64, 5, kU>{});
    case 6: return f(Shape<64, 6, kU>{});
    case 7: case 8: return f(Shape<kU == 4 ? 64 : 512, kU == 4 ? 8 : 1, kU>{});
    default: break;
  }
  if constexpr (kU == 4) {
    if (units <= 640) return f(Shape<64, 10, kU>{});
  }
  switch ((units + 511) / 512) {
    case 1: case 2: return f(Shape<512, 2, kU>{});
    case 3: return f(Shape<512, 3, kU>{});
    case 4: return f(Shape<512, 4, kU>{});
    default: break;
  }
  if constexpr (kU == 4) {
    if (units <= 6 * 512) return f(Shape<512, 6, kU>{});
    return f(Shape<512, 8, kU>{});
  }
  return TM_EINVAL;
}

template <class F>
int with_types(bool x32, bool y32, F&& f) {
  using std::integral_constant;
  if (x32) return y32 ? f(integral_constant<bool, true>{}, integral_constant<bool, true>{})
                      : f(integral_constant<bool, true>{}, integral_constant<bool, false>{});
  return y32 ? f(integral_constant<bool, false>{}, integral_constant<bool, true>{})
             : f(integral_constant<bool, false>{}, integral_constant<bool, false>{});
}

// Workgroups for `rows` rows, `per` of them to each at a time: as many as fill the CUs with `waves` waves each.
int grid_of(int64_t rows, int per, int threads, int waves) {
  const int64_t want = (rows + per - 1) / per, most = static_cast<int64_t>(kCus) * waves * kWave / threads;
  return static_cast<int>(std::min(want, most));
}
// Waves to a CU that the grid is made for (8192 and more rows, each against half and twice as many). Forward: 16 where a
// lane has 8 elements (8192 x 24 heads of 128: 16.0 us, 17.1 with 32), 32 for workgroups of 8 waves with as few (16,384 x 4096: 45.7, 49.5
// with 16), 16 up to 16 elements and 8 past them (8192 x 2560: 15.3, 16.7 with 16). Backward with sums over the rows, whose
// traffic grows with the workgroups: 16 up to 8 elements, 8 up to 24, 4 for one wave's rows past that (8192 x 2560: 32.7 us with the
// sums' launch, 39.8 with 8, 52 with 16; 6001 x 1237 in fp32, 20 elements: 19.7 with 8, 21.3 with 4); without, 8, and 16 for workgroups of 8
// waves (4096 x 9728: 43.5, 53.5 with 8).
template <class S>
int forward_grid(int64_t rows) {
  const int waves = S::kEach > 16 ? 8 : S::kEach > 8 || S::kLanes <= kWave ? 16 : 32;
  return grid_of(rows, S::kForwardThreads / S::kLanes, S::kForwardThreads, waves);
}
template <class S>
int backward_grid(int64_t rows, bool params) {
  const bool one = S::kLanes <= kWave;
  const int waves = S::kEach <= 8 || (!params && !one) ? 16 : params && one && S::kEach > 24 ? 4 : 8;
  return grid_of(rows, S::kBackwardThreads / S::kLanes, S::kBackwardThreads, waves);
}

int backward_grid(int64_t rows, int cols, bool wide, bool params) {
  int grid = 0;
  auto count = [&](auto s) {
    grid = backward_grid<decltype(s)>(rows, params);
    return 0;
  };
  if (wide) with_shape<4>(cols, count);
  else with_shape<8>(cols, count);
  return grid;
}

bool odd(const void* p, bool f32) { return (reinterpret_cast<uintptr_t>(p) & (f32 ? 3 : 1)) != 0; }

int launched(const char* what) {
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? TM_OK : fail(TM_ELAUNCH, "%s: launch failed: %s", what, hipGetErrorString(err));
}

int check_sizes(const char* who, int64_t rows, int64_t cols) {
  if (rows < 0 || rows > (int64_t(1) << 40)) return fail(TM_EINVAL, "%s: rows %lld outside 0..2^40", who, (long long)rows);
  if (cols < 1 || cols > kMaxCols)
    return fail(TM_EINVAL, "%s: cols %lld outside 1..%d", who, (long long)cols, kMaxCols);
  return TM_OK;
}

}  // namespace

extern "C" {

int tm_norm_forward(void* d_y, int y_f32, float* d_rstd, float* d_mean, const void* d_x, int x_f32, int64_t ldx,
                    const void* d_w, int w_f32, const void* d_b, int b_f32, int layer, double eps, int64_t rows, int64_t cols,
                    void* stream) {
  const char* who = "tm_norm_forward";
  if (int rc = check_sizes(who, rows, cols)) return rc;
  if (rows == 0) return TM_OK;
  if (!d_y || !d_x) return fail(TM_EINVAL, "%s: null input or output", who);
  if (layer && d_rstd && !d_mean) return fail(TM_EINVAL, "%s: rstd without mean", who);
  if (ldx < cols && rows > 1) return fail(TM_EINVAL, "%s: rows %lld elements apart", who, (long long)ldx);
  if (odd(d_y, y_f32) || odd(d_x, x_f32) || odd(d_w, w_f32) || odd(d_b, b_f32) || odd(d_rstd, true) || odd(d_mean, true))
    return fail(TM_EINVAL, "%s: a pointer that is not aligned to its elements", who);
  const Forward a = {d_y, d_rstd, d_mean, d_x, d_w, d_b, ldx, rows, static_cast<int>(cols), w_f32, b_f32,
                     static_cast<float>(eps), 1.0f / static_cast<float>(cols)};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int rc = with_types(x_f32, y_f32, [&](auto x32, auto y32) {
    constexpr bool kX = decltype(x32)::value, kY = decltype(y32)::value;
    return with_shape<kX || kY ? 4 : 8>(a.cols, [&](auto shape) {
      using S = decltype(shape);
      const dim3 grid(forward_grid<S>(rows)), block(S::kForwardThreads);
      if (layer) hipLaunchKernelGGL((norm_forward_kernel<S, kX, kY, true>), grid, block, 0, s, a);
      else hipLaunchKernelGGL((norm_forward_kernel<S, kX, kY, false>), grid, block, 0, s, a);
      return TM_OK;
    });
  });
  return rc ? rc : launched(who);
}

size_t tm_norm_workspace_bytes(int64_t rows, int64_t cols, int x_f32, int y_f32, int layer) {
  if (rows < 1 || cols < 1 || cols > kMaxCols) return 0;
  return static_cast<size_t>(backward_grid(rows, static_cast<int>(cols), x_f32 || y_f32, true)) * cols * sizeof(float) * (layer ? 2 : 1);
}

int tm_norm_backward(void* d_dx, void* d_dw, void* d_db, int b_f32, const void* d_dy, int y_f32, int64_t lddy, const void* d_x,
                     int x_f32, int64_t ldx, const float* d_rstd, const float* d_mean, const void* d_w, int w_f32, int dw_f32,
                     int layer, int64_t rows, int64_t cols, void* d_ws, size_t ws_bytes, void* stream) {
  const char* who = "tm_norm_backward";
  if (int rc = check_sizes(who, rows, cols)) return rc;
  if (rows == 0) return fail(TM_EINVAL, "%s: no rows", who);
  if (!d_dy) return fail(TM_EINVAL, "%s: null input", who);
  if ((d_dx || d_dw) && (!d_x || !d_rstd || (layer && !d_mean))) return fail(TM_EINVAL, "%s: null input", who);
  if (!layer && d_db) return fail(TM_EINVAL, "%s: an RMS norm has no bias", who);
  if (!d_dx && !d_dw) d_x = nullptr;
  if (((d_x && ldx < cols) || lddy < cols) && rows > 1)
    return fail(TM_EINVAL, "%s: rows %lld and %lld elements apart", who, (long long)ldx, (long long)lddy);
  if (odd(d_dx, x_f32) || odd(d_dw, dw_f32) || odd(d_db, b_f32) || odd(d_dy, y_f32) || odd(d_x, x_f32) || odd(d_w, w_f32) ||
      odd(d_rstd, true) || odd(d_mean, true))
    return fail(TM_EINVAL, "%s: a pointer that is not aligned to its elements", who);
  const bool params = d_dw || d_db;
  const size_t need = params ? tm_norm_workspace_bytes(rows, cols, x_f32, y_f32, layer) : 0;
  if (ws_bytes < need || (need && (!d_ws || odd(d_ws, true))))
    return fail(TM_EINVAL, "%s: workspace of %zu bytes, %zu needed, aligned to 4", who, d_ws ? ws_bytes : size_t(0), need);
  const int grid = backward_grid(rows, static_cast<int>(cols), x_f32 || y_f32, params);
  float* ws = static_cast<float*>(d_ws);
  Backward a = {d_dx, nullptr, nullptr, d_x, d_dy, d_w, d_rstd, d_mean, ldx, lddy, rows, static_cast<int>(cols), w_f32,
                1.0f / static_cast<float>(cols)};
  if (d_dw) a.dw = ws;
  if (d_db) a.db = ws + static_cast<int64_t>(grid) * cols;
  if (!d_dx && !params) return TM_OK;
  hipStream_t s = static_cast<hipStream_t>(stream);
  int rc = with_types(x_f32, y_f32, [&](auto x32, auto y32) {
    constexpr bool kX = decltype(x32)::value, kY = decltype(y32)::value;
    return with_shape<kX || kY ? 4 : 8>(a.cols, [&](auto shape) {
      using S = decltype(shape);
      const dim3 blocks(grid), block(S::kBackwardThreads);
      if (layer && params) hipLaunchKernelGGL((norm_backward_kernel<S, kX, kY, true, true>), blocks, block, 0, s, a);
      else if (layer) hipLaunchKernelGGL((norm_backward_kernel<S, kX, kY, true, false>), blocks, block, 0, s, a);
      else if (params) hipLaunchKernelGGL((norm_backward_kernel<S, kX, kY, false, true>), blocks, block, 0, s, a);
      else hipLaunchKernelGGL((norm_backward_kernel<S, kX, kY, false, false>), blocks, block, 0, s, a);
      return TM_OK;
    });
  });
  if (rc) return rc;
  if ((rc = launched(who)) || !params) return rc;
  const Join j = {{a.dw, a.db}, {d_dw, d_db}, {dw_f32, b_f32}, grid, a.cols};
  hipLaunchKernelGGL(norm_join_kernel, dim3((a.cols + kWave - 1) / kWave, layer ? 2 : 1), dim3(1024), 0, s, j);
  return launched("norm_join_kernel");
}

}  // extern "C"
