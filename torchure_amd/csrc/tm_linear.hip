// tm_linear.hip -- gfx950 bf16 MFMA products of the linear layers, with what follows them in the
// same kernel: bias, activation, residual and the pre-activation that is kept for the backward pass;
// the gated feed-forward's pair of products and its gradient; the gradients of both operands.
//
//   forward     y   = act(x W^T + b) + r     x rows x inp, W out x inp: both contracted along rows
//                                            of memory ("K-contiguous")
//   gate        h   = silu(x Wg^T) (x Wu^T)  one product over pairs of columns
//   grad_x      dx  = dz W                   W contracted across its rows ("K-major")
//   gate_grad   dh  = dy Wd, then d_gate = dh u silu'(g), d_up = dh silu(g), silu(g) u
//   grad_w      dW  = dz^T x                 both K-major
//
// One kernel template (lin_kernel) with fp32 accumulation on v_mfma_f32_16x16x32_bf16 (the chip's power
// bounds long runs of products, and this shape takes less of it than 32x32x16): 8 wave64, two a
// SIMD, wave (wm, wn) = (w / 4, w % 4) computing 32 kMB x 32 kNB of a 64 kMB x 128 kNB tile. Operands
// stream global -> LDS (global_load_lds, 16 bytes a lane) through five units, each one operand's slice of
// 64 K (32 KB for 256 rows: all of a CU's 160 KB): two hold the current slice, three what comes next, so
// that B's loads have one slice's products to come in and A's two. A K-contiguous operand is loaded in
// whole 128-byte lines (64-byte pieces come in at little more than half the rate: 34 against 56 bytes a
// clock and CU) and lies in 128-byte rows, chunk c of row r at slot c ^ ((r >> 1) & 7); a K-major one in
// whole rows of the tile's columns, chunks swizzled by k_swizzle, and is read transposed
// (ds_read_b64_tr_b16): in both, what a read's lanes get at a time lies on 16 bank groups.
//
// Workgroups are persistent. A workgroup's tiles form one stream of K slices: the loads run ahead of the
// products across tiles, so that a tile starts on operands that came in during the one before it;
// its results leave through the unit used up last, while loads into the others are in flight.
// Workgroup w runs on XCD w % 8; each XCD takes a contiguous range of tile
// positions, in groups of gm x gn tiles whose operand panels share its L2.
//
// Edges: rows and columns past an operand's last are loaded again (their results are not stored); K
// past the operand's end is loaded from 16 bytes of zeros, on both sides, so that no garbage meets
// a zero. Where whole rounds of tiles over the CUs leave some over, or there are few tiles at all, those are
// split over K: fp32 partial tiles in the workspace, added in order by lin_finish_kernel, which then does what
// the unsplit tiles' end does.
//
// Measured (one MI355X, 8192 rows): 8192 -> 8192 805-840 us, 1.31-1.37 PFLOP/s; 9728 -> 2560 with residual 323-335 us, 1.22-1.26;
// 2560 -> 9728 with silu, bias and 8-bit z 386 us, 1.06; the gate 2560 -> 9728 690-720 us, 1.13-1.18; its gradient 540 us
// from bf16, 480 from 8 bits; grad_x of both its products 647 us, 1.26; their grad_w 666 us, 1.23. MFMA busy
// is 62-71% of a launch (39% of the gate's gradient); the rest is ends and first loads.

#include <hip/hip_runtime.h>

#include <stdint.h>

#include <mutex>

#include "torchure_amd.h"
#include "tm_act.h"
#include "tm_internal.h"

namespace {

using tm_act::f32x4;
using tm_act::pack_bf16;
using tm_act::u32x2;
using tm_act::u32x4;
using tm_act::u32x4_at2;
using tm_act::u32x4_at4;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

template <typename... A>
int lin_fail(int code, const char* fmt, A... args) {
  return tm_internal_fail(code, fmt, args...);
}

constexpr int kSliceK = 64;  // K depth of one slice
constexpr int kUnits = 5;    // LDS units, each one operand's slice

constexpr int waitcnt_vm(int n) { return (n & 15) | ((n >> 4) << 14) | (7 << 4) | (15 << 8); }

__device__ const u32x4 g_zeros = {0, 0, 0, 0};  // what K past an operand's end reads

// What follows a product: all of the forward's; only a residual, or nothing; the gate; its gradient.
enum Mode { kLinear, kResidual, kPlain, kGate, kGateGrad };

struct Args {
  const char* a;
  const char* b0;
  const char* b1;           // gate: the up weight; grad_x: the weight of A's second segment
  int64_t a_ld, b_ld;       // bytes from one stored row to the next
  int64_t a_batch;          // bytes from batch 0's A to batch 1's
  int m, n;                 // output rows and columns (gate: features)
  int a_rows, b_rows;       // K-contiguous: rows stored; K-major: columns stored, whole groups of 8
  int ka, kb;               // K that A holds, and that B holds (of one segment)
  int slices, seg;          // K slices, and of them those before b1's (grad_x of two weights)
  int whole, splits, per;   // an XCD's tiles before its split ones; parts of those, of `per` slices each
  int tiles_m, tiles_n, batch, gm, gn, wpx;
  // what follows the product
  char* o0;
  char* o1;                 // batch 1's output; gate_grad: silu(g) u
  int64_t ldo, ldo1;        // elements
  int out_f32, act;
  int n_store;              // columns of an output row that are written (past n: zeros)
  const char* bias;
  const char* res;
  int64_t ldr;
  int bias_f32, res_f32;
  char* z0;                 // pre-activations (gate products), up products
  char* z1;
  uint8_t* s0;              // their block exponents, where they are held as e4m3
  uint8_t* s1;
  int64_t ldz;
  int held, blocks;         // TM_HELD_*; blocks of 32 columns in a row of exponents
  float* partial;
};

// Chunk c of K row `row` of a K-major operand lies at slot c ^ k_swizzle(row): what 32 lanes read at a time,
// 2 chunks of 8 K rows (4 in a row, and 4 that are 8 on), then falls on 16 different bank groups. Rows
// of 192 columns are 384 bytes, so that odd ones are half the banks on already, and have 3 times 8 chunks.
template <int kT>
__device__ __forceinline__ int k_swizzle(int row) {
  if constexpr (kT == 192) return (row & 2) | (row >> 3 & 1) << 2;
  else return 2 * ((row & 3) | (row >> 3 & 1) << 2);
}

// ------------------------------------------------------------------------------ a tile's results
//
// A wave's accumulators come out in blocks of 32 x 32, each 2 x 2 of the products' 16 x 16: there lane l
// holds row l % 16, columns 4 (l / 16) .. + 3. Each block goes through this wave's strip of LDS (fp32, 128-byte rows, chunk c of
// row r at slot c ^ ((r >> 1) & 7): a wave's LDS accesses are served in order, so no barrier and no wait
// is needed between its writes and its reads) and is read back in the order of the output's rows: lane l
// has columns 8 (l % 4) .. + 7 of rows l / 4 and 16 + l / 4. From there on every access to memory is 16
// bytes a lane and whole pieces of rows, whatever is fused, and one copy of the code serves all blocks.

typedef const __attribute__((address_space(4))) Args* ArgsPtr;  // the kernel's arguments, where they are

// What a tile's end needs of them, in scalar registers: read once for each tile and before its first block (one
// after the other as a block needs them, the reads' latencies were 10 us of a tile; kept through
// the products, they spill).
struct End {
  int m;
  int n;
  char* o0;
  char* o1;
  int64_t ldo;
  int64_t ldo1;
  int out_f32;
  int act;
  int n_store;
  const char* bias;
  const char* res;
  int64_t ldr;
  int bias_f32;
  int res_f32;
  char* z0;
  char* z1;
  uint8_t* s0;
  uint8_t* s1;
  int64_t ldz;
  int held;
  int blocks;
};

template <int kMode>
__device__ __forceinline__ End end_of() {
  ArgsPtr g = (ArgsPtr)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(g));
  End e = {};
#define TM_TAKE(field) e.field = g->field
  if constexpr (kMode == kLinear) {
    TM_TAKE(m); TM_TAKE(n); TM_TAKE(o0); TM_TAKE(ldo); TM_TAKE(out_f32); TM_TAKE(act);
    TM_TAKE(bias); TM_TAKE(res); TM_TAKE(ldr); TM_TAKE(bias_f32); TM_TAKE(res_f32);
    TM_TAKE(z0); TM_TAKE(s0); TM_TAKE(ldz); TM_TAKE(held); TM_TAKE(blocks);
  }
  if constexpr (kMode == kResidual) {
    TM_TAKE(m); TM_TAKE(n); TM_TAKE(o0); TM_TAKE(ldo); TM_TAKE(out_f32); TM_TAKE(res);
    TM_TAKE(ldr); TM_TAKE(res_f32);
  }
  if constexpr (kMode == kPlain) {
    TM_TAKE(m); TM_TAKE(n); TM_TAKE(o0); TM_TAKE(o1); TM_TAKE(ldo); TM_TAKE(out_f32);
  }
  if constexpr (kMode == kGate) {
    TM_TAKE(m); TM_TAKE(n); TM_TAKE(n_store); TM_TAKE(o0); TM_TAKE(ldo); TM_TAKE(z0); TM_TAKE(z1);
    TM_TAKE(s0); TM_TAKE(s1); TM_TAKE(ldz); TM_TAKE(held); TM_TAKE(blocks);
  }
  if constexpr (kMode == kGateGrad) {
    TM_TAKE(m); TM_TAKE(n); TM_TAKE(n_store); TM_TAKE(o0); TM_TAKE(o1); TM_TAKE(ldo); TM_TAKE(ldo1);
    TM_TAKE(z0); TM_TAKE(z1); TM_TAKE(s0); TM_TAKE(s1); TM_TAKE(ldz); TM_TAKE(held); TM_TAKE(blocks);
  }
#undef TM_TAKE
#define TM_KEEP(field) asm volatile("" : "+s"(e.field))
  if constexpr (kMode == kLinear) {
    TM_KEEP(m); TM_KEEP(n); TM_KEEP(o0); TM_KEEP(ldo); TM_KEEP(out_f32); TM_KEEP(act);
    TM_KEEP(bias); TM_KEEP(res); TM_KEEP(ldr); TM_KEEP(bias_f32); TM_KEEP(res_f32);
    TM_KEEP(z0); TM_KEEP(s0); TM_KEEP(ldz); TM_KEEP(held); TM_KEEP(blocks);
  }
  if constexpr (kMode == kResidual) {
    TM_KEEP(m); TM_KEEP(n); TM_KEEP(o0); TM_KEEP(ldo); TM_KEEP(out_f32); TM_KEEP(res);
    TM_KEEP(ldr); TM_KEEP(res_f32);
  }
  if constexpr (kMode == kPlain) {
    TM_KEEP(m); TM_KEEP(n); TM_KEEP(o0); TM_KEEP(o1); TM_KEEP(ldo); TM_KEEP(out_f32);
  }
  if constexpr (kMode == kGate) {
    TM_KEEP(m); TM_KEEP(n); TM_KEEP(n_store); TM_KEEP(o0); TM_KEEP(ldo); TM_KEEP(z0); TM_KEEP(z1);
    TM_KEEP(s0); TM_KEEP(s1); TM_KEEP(ldz); TM_KEEP(held); TM_KEEP(blocks);
  }
  if constexpr (kMode == kGateGrad) {
    TM_KEEP(m); TM_KEEP(n); TM_KEEP(n_store); TM_KEEP(o0); TM_KEEP(o1); TM_KEEP(ldo); TM_KEEP(ldo1);
    TM_KEEP(z0); TM_KEEP(z1); TM_KEEP(s0); TM_KEEP(s1); TM_KEEP(ldz); TM_KEEP(held); TM_KEEP(blocks);
  }
#undef TM_KEEP
  return e;
}

template <bool kV>
struct Bool {
  static constexpr bool value = kV;
};

struct Block {
  float v[16];  // [row half][column]
};

// A lane's places: where it writes and reads a block in the strip, and its bytes past a block's first element
// in each matrix (rows 16 on: 16 rows more).
struct Lane {
  uint32_t w[2], r[2];
  uint32_t out, out1, res, z;
};

template <int kMode>
__device__ __forceinline__ Lane lane_of(const End& g, uint32_t stg, int lane) {
  Lane l;
  const uint32_t row = lane & 15, r = lane >> 2, sr = (r >> 1) & 7, c = 2 * (lane & 3), col = 8 * (lane & 3);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    l.w[i] = stg + row * 128 + (((4 * i + (lane >> 4)) ^ (row >> 1)) << 4);
    l.r[i] = stg + r * 128 + (((c + i) ^ sr) << 4);
  }
  l.out = (r * static_cast<uint32_t>(g.ldo) + col) * (kMode <= kPlain && g.out_f32 ? 4 : 2);
  if constexpr (kMode <= kResidual) l.res = (r * static_cast<uint32_t>(g.ldr) + col) * (g.res_f32 ? 4 : 2);
  if constexpr (kMode == kGateGrad) l.out1 = (r * static_cast<uint32_t>(g.ldo1) + col) * 2;
  if constexpr (kMode == kLinear || kMode >= kGate) l.z = (r * static_cast<uint32_t>(g.ldz) + col) * (g.held == TM_HELD_BF16 ? 2 : 1);
  return l;
}

// kHalves: a strip of 2 KB, 16 rows at a time (else 4 KB). acc[row half][column half].
template <bool kHalves>
__device__ __forceinline__ void to_rows(Block& b, const f32x4 (&acc)[2][2], const Lane& l) {
  auto write = [&](int h, int at) {  // 16 rows on: the same slots
#pragma unroll
    for (int i = 0; i < 2; ++i)
      asm volatile("ds_write_b128 %0, %1 offset:%2" ::"v"(l.w[i]), "v"(acc[h][i]), "i"(at) : "memory");
  };
  auto keep = [&](int at, const f32x4& t) {
    b.v[at] = t.x;
    b.v[at + 1] = t.y;
    b.v[at + 2] = t.z;
    b.v[at + 3] = t.w;
  };
  f32x4 t[4];
  if constexpr (kHalves) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      write(h, 0);
      asm volatile("ds_read_b128 %0, %2\n\tds_read_b128 %1, %3\n\ts_waitcnt lgkmcnt(0)"
                   : "=&v"(t[0]), "=&v"(t[1])
                   : "v"(l.r[0]), "v"(l.r[1])
                   : "memory");
      keep(8 * h, t[0]);
      keep(8 * h + 4, t[1]);
    }
  } else {
    write(0, 0);
    write(1, 2048);
    asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %1, %5\n\tds_read_b128 %2, %4 offset:2048\n\t"
                 "ds_read_b128 %3, %5 offset:2048\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(t[0]), "=&v"(t[1]), "=&v"(t[2]), "=&v"(t[3])
                 : "v"(l.r[0]), "v"(l.r[1])
                 : "memory");
#pragma unroll
    for (int i = 0; i < 4; ++i) keep(4 * i, t[i]);
  }
}

// Eight bf16 or fp32 values as they lie in memory.
struct Raw8 {
  u32x4 w[2];
};

// What is at p is in memory: the compiler cannot tell from a pointer that the kernel's arguments hold, and its
// flat accesses would count as LDS accesses too, which the strip's reads wait for.
template <typename T>
__device__ __forceinline__ __attribute__((address_space(1))) T* mem(const void* p) {
  return (__attribute__((address_space(1))) T*)reinterpret_cast<uintptr_t>(p);
}

// Rows may start at any element: an access of 16 bytes need not be aligned to them. (1237 x 777 -> 1001 with
// a residual, whose rows are odd: 15.4 us so, 21.5 us with an access an element.) No branch: where two ways of
// loading meet, the loads are waited for, early or not.
__device__ __forceinline__ Raw8 raw8(const char* p, bool f32) {
  return {{*mem<u32x4_at2>(p), *mem<u32x4_at2>(p + (f32 ? 16 : 0))}};
}

__device__ __forceinline__ Raw8 raw8(const char* p, bool f32, int left) {  // `left` of them exist
  if (left >= 8) return raw8(p, f32);
  uint32_t w[8] = {};
#pragma unroll
  for (int e = 0; e < 7; ++e)
    if (e < left) {
      if (f32) w[e] = mem<uint32_t>(p)[e];
      else w[e / 2] |= static_cast<uint32_t>(mem<uint16_t>(p)[e]) << (16 * (e & 1));
    }
  return {{u32x4{w[0], w[1], w[2], w[3]}, u32x4{w[4], w[5], w[6], w[7]}}};
}

__device__ __forceinline__ void values8(float* x, const Raw8& r, bool f32) {
  const uint32_t a[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w}, b[4] = {r.w[1].x, r.w[1].y, r.w[1].z, r.w[1].w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (f32) {
      x[e] = __uint_as_float(a[e]);
      x[4 + e] = __uint_as_float(b[e]);
    } else {
      x[2 * e] = tm_act::bf16_lo(a[e]);
      x[2 * e + 1] = tm_act::bf16_hi(a[e]);
    }
  }
}

__device__ __forceinline__ void put8(char* p, const float* x, bool f32) {
  if (f32) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      mem<u32x4_at4>(p)[h] = u32x4{__float_as_uint(x[4 * h]), __float_as_uint(x[4 * h + 1]), __float_as_uint(x[4 * h + 2]),
                                   __float_as_uint(x[4 * h + 3])};
  } else {
    *mem<u32x4_at2>(p) =
        u32x4{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7])};
  }
}

__device__ __forceinline__ void put8(char* p, const float* x, bool f32, int left) {
  if (left >= 8) return put8(p, x, f32);
#pragma unroll
  for (int e = 0; e < 7; ++e)
    if (e < left) {
      if (f32) mem<float>(p)[e] = x[e];
      else mem<uint16_t>(p)[e] = static_cast<uint16_t>(pack_bf16(x[e], 0.0f));
    }
}

// Where a block is, and which of a lane's values exist (kWhole: all).
struct Spot {
  int m0, n0;
  int cols;     // columns left from the lane's first
  bool row[2];
};

__device__ __forceinline__ Spot spot_of(const End& g, int m0, int n0, int lane) {
  const int m = m0 + (lane >> 2);
  return {m0, n0, g.n - n0 - 8 * (lane & 3), {m < g.m, m + 16 < g.m}};
}

// A block's first element, row half i, of a matrix with rows ld elements of `size` bytes apart.
__device__ __forceinline__ char* at_block(const char* p, int64_t ld, int size, const Spot& s, int i) {
  return const_cast<char*>(p) + ((static_cast<int64_t>(s.m0) + 16 * i) * ld + s.n0) * size;
}

__device__ __forceinline__ void mask(Block& b, const Spot& s) {
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (!s.row[i / 8] || i % 8 >= s.cols) b.v[i] = 0.0f;
}

__device__ __forceinline__ int64_t exponent_at(const End& g, const Spot& s) {
  return static_cast<int64_t>(s.m0 >> 5) * g.blocks + (s.n0 >> 5);
}

// A block as the backward pass reads it (its values outside the matrix zero): the padding columns are written
// too.
template <bool kWhole>
__device__ __forceinline__ void hold(const End& g, const Lane& l, const Block& b, const Spot& s, char* z, uint8_t* exps,
                                     int lane) {
  if (g.held == TM_HELD_BF16) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (kWhole || (s.row[i] && s.n0 + 8 * (lane & 3) < g.ldz))
        put8(at_block(z, g.ldz, 2, s, i) + l.z, b.v + 8 * i, false);
  } else {
    auto encode = [&](uint32_t most, auto any) {
      const int e = tm_act::block_exponent(most);
      const float inv = tm_act::two_to(-e);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float* x = b.v + 8 * i;
        const u32x2 w = {tm_act::encode4<decltype(any)::value>(x[0], x[1], x[2], x[3], inv),
                         tm_act::encode4<decltype(any)::value>(x[4], x[5], x[6], x[7], inv)};
        if (kWhole || s.row[i]) *mem<u32x2>(at_block(z, g.ldz, 1, s, i) + l.z) = w;
      }
      if (lane == 0) *mem<uint8_t>(exps + exponent_at(g, s)) = static_cast<uint8_t>(e + 127);
    };
    const uint32_t most = tm_act::wave_max(tm_act::largest<16>(b.v));
    if (most < tm_act::kPlainMost) encode(most, Bool<false>{});
    else encode(tm_act::wave_max(tm_act::largest_finite<16>(b.v)), Bool<true>{});
  }
}

// What a block's end reads from memory: the residual, or the gate's and up's products. (Whole tiles' is read
// while the block before it is worked on.)
struct Early {
  Raw8 a[2], b[2];  // [row half]
  uint32_t exps[2];
};

template <int kMode, bool kWhole>
__device__ __forceinline__ Early early_of(const End& g, const Lane& l, int m0, int n0, int lane) {
  Early r = {};
  if (!kWhole && (m0 >= g.m || n0 >= g.n)) return r;
  const Spot s = spot_of(g, m0, n0, lane);
  if constexpr (kMode <= kResidual) {
    const int size = g.res_f32 ? 4 : 2;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const char* p = at_block(g.res, g.ldr, size, s, i);
      if (kWhole) r.a[i] = raw8(p + l.res, g.res_f32);
      else if (s.row[i] && s.cols > 0)
        r.a[i] = raw8(p + l.res, g.res_f32, s.cols);
    }
  }
  if constexpr (kMode == kGateGrad) {
    const bool bf16 = g.held == TM_HELD_BF16;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (!kWhole && !(s.row[i] && (!bf16 || s.n0 + 8 * (lane & 3) < g.ldz))) continue;
      const char *pg = at_block(g.z0, g.ldz, bf16 ? 2 : 1, s, i), *pu = at_block(g.z1, g.ldz, bf16 ? 2 : 1, s, i);
      auto load = [&](const char* p) {
        const u32x2 x = *mem<u32x2>(p), y = *mem<u32x2>(p + (bf16 ? 8 : 0));
        return u32x4{x.x, x.y, y.x, y.y};
      };
      r.a[i].w[0] = load(pg + l.z);
      r.b[i].w[0] = load(pu + l.z);
    }
    const char *p0 = bf16 ? g.z0 : reinterpret_cast<const char*>(g.s0), *p1 = bf16 ? g.z1 : reinterpret_cast<const char*>(g.s1);
    const int64_t at = bf16 ? 0 : exponent_at(g, s);
    r.exps[0] = *mem<uint8_t>(p0 + at);
    r.exps[1] = *mem<uint8_t>(p1 + at);
  }
  return r;
}

template <bool kWhole>
__device__ __forceinline__ void add_residual(const End& g, Block& b, const Early& early) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float x[8];
    values8(x, early.a[i], g.res_f32);
#pragma unroll
    for (int e = 0; e < 8; ++e) b.v[8 * i + e] += x[e];
  }
}

// y = act(z + b) + r, and z as it is kept. The products' fp32 sums are rounded once, in y's type; z
// is rounded to what the backward pass reads.
template <bool kWhole>
__device__ __forceinline__ void end_linear(const End& g, const Lane& l, Block& b, const Spot& s, const Raw8& bias,
                                           int lane) {
  if (g.bias) {
    float x[8];
    values8(x, bias, g.bias_f32);
#pragma unroll
    for (int i = 0; i < 16; ++i) b.v[i] += x[i % 8];
  }
  if (g.held) {
    if (!kWhole) mask(b, s);
    hold<kWhole>(g, l, b, s, g.z0, g.s0, lane);
  }
  const int act = g.act;
  auto each = [&](auto f) {
#pragma unroll
    for (int i = 0; i < 16; ++i) b.v[i] = f(b.v[i]);
  };
  if (act == tm_act::kRelu) each([](float z) { return tm_act::act1(tm_act::kRelu, z); });
  else if (act == tm_act::kSilu) each([](float z) { return tm_act::act1(tm_act::kSilu, z); });
  else if (act == tm_act::kGelu) each([](float z) { return tm_act::act1(tm_act::kGelu, z); });
  else if (act == tm_act::kGeluTanh) each([](float z) { return tm_act::act1(tm_act::kGeluTanh, z); });
  if (g.res) {  // read here, not early: the registers are the activation's
    if (kWhole) add_residual<true>(g, b, early_of<kLinear, true>(g, l, s.m0, s.n0, lane));
    else add_residual<false>(g, b, early_of<kLinear, false>(g, l, s.m0, s.n0, lane));
  }
}

// A block of y, of a gradient: kWhole, in 16-byte pieces.
template <bool kWhole>
__device__ __forceinline__ void store_block(const End& g, const Lane& l, char* out, const Block& b, const Spot& s, int lane) {
  const int size = g.out_f32 ? 4 : 2;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    char* p = at_block(out, g.ldo, size, s, i);
    if (kWhole) put8(p + l.out, b.v + 8 * i, g.out_f32);
    else if (s.row[i] && s.cols > 0) put8(p + l.out, b.v + 8 * i, g.out_f32, s.cols);
  }
}

// h = silu(g) u of 32 features, g and u kept on the way. Columns of padding are zeros.
template <bool kWhole>
__device__ __forceinline__ void end_gate(const End& g, const Lane& l, Block& gate, Block& up, const Spot& s, int lane) {
  if (!kWhole) {
    mask(gate, s);
    mask(up, s);
  }
  if (g.held && s.n0 < g.n) {
    hold<kWhole>(g, l, gate, s, g.z0, g.s0, lane);
    hold<kWhole>(g, l, up, s, g.z1, g.s1, lane);
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) gate.v[i] = gate.v[i] * tm_act::sigmoid(gate.v[i]) * up.v[i];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (kWhole || (s.row[i] && s.n0 + 8 * (lane & 3) < g.n_store))
      put8(at_block(g.o0, g.ldo, 2, s, i) + l.out, gate.v + 8 * i, false);
}

// From dh: d_gate and d_up (columns 0.. and n_store.. of o0's rows) and silu(g) u (o1), g and u as held.
template <bool kWhole>
__device__ __forceinline__ void end_gate_grad(const End& g, const Lane& l, Block& d, const Spot& s, const Early& early,
                                              int lane) {
  if (!kWhole && s.n0 + 32 > g.n) mask(d, s);  // g and u are zero there
  const bool bf16 = g.held == TM_HELD_BF16;
  float sg = 1.0f, su = 1.0f;
  if (!bf16 && s.n0 < g.n) {
    sg = tm_act::two_to(static_cast<int>(early.exps[0]) - 127);
    su = tm_act::two_to(static_cast<int>(early.exps[1]) - 127);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float z[8], u[8];
    if (bf16) {
      values8(z, early.a[i], false);
      values8(u, early.b[i], false);
    } else {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const f32x4 x = tm_act::decode4(e ? early.a[i].w[0].y : early.a[i].w[0].x, sg);
        const f32x4 y = tm_act::decode4(e ? early.b[i].w[0].y : early.b[i].w[0].x, su);
        z[4 * e] = x.x; z[4 * e + 1] = x.y; z[4 * e + 2] = x.z; z[4 * e + 3] = x.w;
        u[4 * e] = y.x; u[4 * e + 1] = y.y; u[4 * e + 2] = y.z; u[4 * e + 3] = y.w;
      }
    }
    float* dh = d.v + 8 * i;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float q = tm_act::sigmoid(z[e]), a = z[e] * q;
      z[e] = dh[e] * u[e] * tm_act::silu_grad(z[e], q);
      dh[e] *= a;
      u[e] *= a;
    }
    if (kWhole || (s.row[i] && s.n0 + 8 * (lane & 3) < g.n_store)) {
      char* o = at_block(g.o0, g.ldo, 2, s, i);
      put8(o + l.out, z, false);
      put8(o + static_cast<int64_t>(g.n_store) * 2 + l.out, dh, false);
      if (g.o1) put8(at_block(g.o1, g.ldo1, 2, s, i) + l.out1, u, false);
    }
    __builtin_amdgcn_sched_barrier(0);  // one half's values at a time
  }
}

template <int kMode, bool kWhole>
__device__ __forceinline__ void end_block(const End& g, const Lane& l, int batch, Block& x, Block& y, int m, int n,
                                          const Raw8& bias, const Early& early, int lane) {
  const Spot s = spot_of(g, m, n, lane);
  if constexpr (kMode == kLinear) end_linear<kWhole>(g, l, x, s, bias, lane);
  if constexpr (kMode == kResidual) add_residual<kWhole>(g, x, early);
  if constexpr (kMode <= kPlain) store_block<kWhole>(g, l, kMode == kPlain && batch ? g.o1 : g.o0, x, s, lane);
  else if constexpr (kMode == kGate) end_gate<kWhole>(g, l, x, y, s, lane);
  else end_gate_grad<kWhole>(g, l, x, s, early, lane);
}

// A wave's blocks, of which the first is at row m0, column n0, down each column of blocks. Of tiles inside the
// matrix, one after the other in straight code (but for kLinear, whose code is long); else in a loop whose
// first step picks the block's registers. No register may spill here: a spill's reload waits for all
// stores before it.
// kNarrow: of the one block's columns the first 16.
template <int kMode, bool kHalves, int kRowBlocks, int kColBlocks, bool kNarrow = false>
__device__ __forceinline__ void finish(f32x4 (&acc)[2 * kRowBlocks][2 * kColBlocks], int batch, int m0, int n0, int lane,
                                       uint32_t stg) {
  End g = end_of<kMode>();
  if (kNarrow) {
    g.n = min(g.n, n0 + 16);
    if (kMode == kGate) g.n_store = min(g.n_store, n0 + 16);
  }
  asm volatile("" : "+v"(lane));  // what derives from it is made again for each tile: kept, it spills
  const Lane l = lane_of<kMode>(g, stg, lane);
  constexpr int kPer = kMode == kGate ? 2 : 1, kCols = kColBlocks / kPer, kBlocks = kRowBlocks * kCols;
  constexpr bool kReads = kMode == kResidual || kMode == kGateGrad;
  const bool whole = m0 + 32 * kRowBlocks <= g.m && n0 + 32 * kCols <= g.n;
  auto pick = [&](Block& x, Block& y, int c) {
    const int jj = 2 * (c % kRowBlocks), ii = 2 * kPer * (c / kRowBlocks);
    const f32x4 t[2][2] = {{acc[jj][ii], acc[jj][ii + 1]}, {acc[jj + 1][ii], acc[jj + 1][ii + 1]}};
    to_rows<kHalves>(x, t, l);
    if constexpr (kMode == kGate) {
      const f32x4 u[2][2] = {{acc[jj][ii + 2], acc[jj][ii + 3]}, {acc[jj + 1][ii + 2], acc[jj + 1][ii + 3]}};
      to_rows<kHalves>(y, u, l);
    }
  };
  if (kMode != kLinear && whole) {
    Early early;
    if constexpr (kReads) early = early_of<kMode, true>(g, l, m0, n0, lane);
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      Block x, y;
      pick(x, y, b);
      const Early now = early;
      if (kReads && b + 1 < kBlocks)
        early = early_of<kMode, true>(g, l, m0 + (b + 1) % kRowBlocks * 32, n0 + (b + 1) / kRowBlocks * 32, lane);
      end_block<kMode, true>(g, l, batch, x, y, m0 + b % kRowBlocks * 32, n0 + b / kRowBlocks * 32, Raw8{}, now, lane);
      __builtin_amdgcn_sched_barrier(0);
    }
    return;
  }
  Raw8 bias = {};
#pragma unroll 1
  for (int b = 0; b < kBlocks; ++b) {
    const int m = m0 + b % kRowBlocks * 32, n = n0 + b / kRowBlocks * 32;
    if (m >= g.m || n >= (kMode >= kGate ? g.n_store : g.n)) continue;
    if constexpr (kMode == kLinear)
      if (g.bias && b % kRowBlocks == 0)
        bias = raw8(g.bias + (static_cast<int64_t>(n) + 8 * (lane & 3)) * (g.bias_f32 ? 4 : 2), g.bias_f32,
                    g.n - n - 8 * (lane & 3));
    Early early = {};
    if constexpr (kReads) early = early_of<kMode, false>(g, l, m, n, lane);
    Block x, y;
#pragma unroll
    for (int c = 0; c < kBlocks; ++c)
      if (b == c) pick(x, y, c);
    if (kMode == kLinear && whole) end_block<kMode, kMode == kLinear>(g, l, batch, x, y, m, n, bias, early, lane);
    else end_block<kMode, false>(g, l, batch, x, y, m, n, bias, early, lane);
  }
  // vmcnt(0): else the slices' loop may wait in every slice for a load whose use a branch here has passed by.
  __builtin_amdgcn_s_waitcnt(0x0f70);
}

// ------------------------------------------------------------------------------ the product

template <int kMB, int kNB>
struct Tile {
  static constexpr int kTM = 64 * kMB, kTN = 128 * kNB;
  static constexpr int kUnit = (kTM > kTN ? kTM : kTN) * kSliceK * 2;  // LDS for one operand's slice
  static constexpr int kStrip = kUnit / 8 < 4096 ? 2048 : 4096;        // one wave's, in a unit just used up
  static constexpr bool kHalves = kStrip == 2048;
  static constexpr int kLds = kUnits * kUnit;  // 80 KB (two workgroups a CU) or 160 KB
};

// a / d and the remainder, for 0 <= a < 2^22: the estimate is off by at most one.
__device__ __forceinline__ int divide(int a, int d, int& rem) {
  int q = static_cast<int>(static_cast<float>(a) * __builtin_amdgcn_rcpf(static_cast<float>(d)));
  rem = a - q * d;
  if (rem < 0) {
    --q;
    rem += d;
  } else if (rem >= d) {
    ++q;
    rem -= d;
  }
  return q;
}

// An XCD's share of the tiles: `whole` of them in one position each, then the others in g.splits positions each,
// all first parts before all second ones.
struct Share {
  int first, whole, others;
  __device__ __forceinline__ int positions(const Args& g) const { return whole + others * g.splits; }
};

__device__ __forceinline__ Share share_of(const Args& g, int xcd) {
  const int T = g.tiles_m * g.tiles_n * g.batch, t8 = (T + 7) / 8, first = xcd * t8;
  const int n = max(0, min(t8, T - first)), whole = min(g.whole, n);
  return {first, whole, n - whole};
}

// Tile -> batch and the tile's first row and column (gate: feature): n-blocks of gn tile columns; inside each,
// m-blocks of gm tile rows, a block's gm x gn tiles consecutive.
template <int kTM, int kTN, bool kHalf>
__device__ __forceinline__ void place(const Args& g, int tile, int& batch, int& m0, int& n0) {
  batch = 0;
  if (g.batch > 1) batch = divide(tile, g.tiles_m * g.tiles_n, tile);
  int rem, tn;
  const int nb = divide(tile, g.tiles_m * g.gn, rem);
  const int gn = min(g.gn, g.tiles_n - nb * g.gn);
  const int mb = divide(rem, g.gm * gn, rem);
  const int tm = mb * g.gm + divide(rem, gn, tn);
  m0 = tm * kTM;
  n0 = (nb * g.gn + tn) * (kHalf ? kTN / 2 : kTN);
}

// An XCD's position -> tile, and its slices [lit, lend); the part of a split tile, else -1.
__device__ __forceinline__ int part_of(const Args& g, const Share& s, int p, int& tile, int& lit, int& lend) {
  lit = 0;
  lend = g.slices;
  tile = s.first + p;
  if (p < s.whole) return -1;
  int rem;
  const int part = divide(p - s.whole, s.others, rem);
  tile = s.first + s.whole + rem;
  lit = part * g.per;
  lend = min(lit + g.per, g.slices);
  return part;
}

// Where part `part` of an XCD's split tile `tile` lies in the workspace, in tiles.
__device__ __forceinline__ int64_t partial_at(const Args& g, int tile, int part) {
  const int T = g.tiles_m * g.tiles_n * g.batch, t8 = (T + 7) / 8, xcd = tile / t8;
  return static_cast<int64_t>(xcd * (t8 - g.whole) + tile - xcd * t8 - g.whole) * g.splits + part;
}

// One operand's loads: a stream of units (the tile's kT rows or columns of 64 K) over the workgroup's
// positions. Load j of wave w fills KB 8 j + w: K-contiguous, 8 rows of 128 bytes; K-major, whole K rows of
// the tile's columns.
template <int kT, bool kContig, bool kIsA, bool kPairs, bool kRagged, int kTM, int kTN>
struct Feed {
  static constexpr int kLoads = kT / 64;
  int lp, lit, lend;      // position; slice of the next one that is not plain; the position's last, + 1
  int plain;              // slices before that: one after another, whole
  const char* at;         // the operand at the next slice
  int64_t step, col;
  uint32_t off[kLoads];   // this lane's bytes past `at`

  // the operand's row (or K row) and 16-byte chunk that a lane loads in KB q
  static __device__ __forceinline__ void spot(int lane, int q, int& r, int& c) {
    if constexpr (kContig) {
      r = q * 8 + lane / 8;
      c = (lane % 8) ^ ((r >> 1) & 7);
    } else {
      const int id = q * 64 + lane;
      r = id / (kT / 8);
      c = id % (kT / 8) ^ k_swizzle<kT>(r);
    }
  }
  __device__ __forceinline__ int left(const Args& g) const {  // K that the operand holds from slice lit on
    if constexpr (kIsA) return g.ka - lit * kSliceK;
    else return g.kb - (!kContig && lit >= g.seg ? lit - g.seg : lit) * kSliceK;
  }
  __device__ __forceinline__ void count(const Args& g) {
    int n = lend - 1 - lit;
    if (kRagged) n = min(n, left(g) / kSliceK);
    if (!kIsA && !kContig && lit < g.seg) n = min(n, g.seg - 1 - lit);
    plain = max(n, 0);
    lit += plain;
  }
  __device__ __forceinline__ void seek(const Args& g, const Share& sh, int pos, int lane, int wave) {
    asm volatile("" : "+v"(lane));  // derived again for each tile, not kept through the products
    int tile, batch, m0, n0;
    lp = pos;
    part_of(g, sh, pos, tile, lit, lend);
    place<kTM, kTN, kPairs>(g, tile, batch, m0, n0);
    const int64_t ld = kIsA ? g.a_ld : g.b_ld;
    step = kContig ? kSliceK * 2 : kSliceK * ld;
    if constexpr (kIsA) {
      at = kContig ? g.a + m0 * ld + lit * step : g.a + batch * g.a_batch + static_cast<int64_t>(m0) * 2 + lit * step;
    } else if constexpr (kContig) {
      at = (kPairs && (wave & 4) ? g.b1 : g.b0) + n0 * ld + lit * step;  // KB 8 j + 4 .. 7: the up weight's rows
    } else {
      col = static_cast<int64_t>(n0) * 2;
      at = lit >= g.seg ? g.b1 + col + (lit - g.seg) * step : g.b0 + col + lit * step;
    }
    const int most = kIsA ? g.a_rows - m0 : g.b_rows - n0;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      int r, c;
      spot(lane, 8 * j + wave, r, c);
      if constexpr (kContig) {
        const int row = kPairs && !kIsA ? (r >> 6) * 32 + (r & 31) : r;
        off[j] = static_cast<uint32_t>(min(row, most - 1)) * static_cast<uint32_t>(ld) + c * 16;
      } else {
        off[j] = static_cast<uint32_t>(r) * static_cast<uint32_t>(ld) + min(8 * c, most - 8) * 2;
      }
    }
  }
  static __device__ __forceinline__ void to_lds(const char* from, uint8_t* unit, int j) {
    __builtin_amdgcn_global_load_lds((const void __attribute__((address_space(1)))*)from,
                                     (void __attribute__((address_space(3)))*)(unit + j * 8192), 16, 0, 0);
  }
  // `unit` is where this wave's first KB goes
  __device__ __forceinline__ void load(uint8_t* unit, int j) const { to_lds(at + off[j], unit, j); }
  __device__ __forceinline__ void next() {
    at += step;
    --plain;
  }
  // The slice that is not plain: the position's last, or one that reaches past the operand's K (zeros) or
  // up to its other segment.
  __device__ __forceinline__ void load_event(const Args& g, const Share& sh, uint8_t* unit, int lane, int wave) {
    const int k = kRagged ? left(g) : kSliceK;
    if (k >= kSliceK) {
#pragma unroll
      for (int j = 0; j < kLoads; ++j) load(unit, j);
    } else {
      int ln = lane;
      asm volatile("" : "+v"(ln));
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        int r, c;
        spot(ln, 8 * j + wave, r, c);
        to_lds((kContig ? c * 8 : r) < k ? at + off[j] : reinterpret_cast<const char*>(&g_zeros), unit, j);
      }
    }
    past_event(g, sh, lane, wave);
  }
  // On from the slice that is not plain.
  __device__ __forceinline__ void past_event(const Args& g, const Share& sh, int lane, int wave) {
    if (lit + 1 < lend) {
      ++lit;
      at += step;
      if (!kIsA && !kContig && lit == g.seg) at = g.b1 + col;
    } else if (lp + g.wpx < sh.positions(g)) {
      seek(g, sh, lp + g.wpx, lane, wave);
    }  // else: the last slice again, which nothing reads
    count(g);
  }
  __device__ __forceinline__ void load_all(const Args& g, const Share& sh, uint8_t* unit, int lane, int wave) {
    if (plain > 0) {
#pragma unroll
      for (int j = 0; j < kLoads; ++j) load(unit, j);
      next();
    } else {
      load_event(g, sh, unit, lane, wave);
    }
  }
};

template <int kQ>
struct Quarter {
  static constexpr int q = kQ;
};

template <int kMB, int kNB, bool kAK, bool kBK, bool kRagged, int kMode>
__global__ __launch_bounds__(512, kMB * kNB == 2 ? 4 : 2) void lin_kernel(const Args g) {
  using C = Tile<kMB, kNB>;
  constexpr int kTM = C::kTM, kTN = C::kTN, kUnit = C::kUnit;
  constexpr int kFB = 2 * kNB;  // B fragments, 16 columns each; A: two halves of kMB, 16 rows each
  constexpr int kRdA = kAK ? kMB : 2 * kMB, kRdB = kBK ? kFB : 2 * kFB;
  constexpr bool kPairs = kMode == kGate;
  static_assert(!kPairs || (kNB == 2 && kBK), "gate and up columns alternate by 32 within a wave");
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const Share sh = share_of(g, static_cast<int>(blockIdx.x % 8));
  const int pend = sh.positions(g);
  int p = static_cast<int>(blockIdx.x / 8);
  if (p >= pend) return;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 2, wn = wave & 3;

  // ---- fragments of v_mfma_f32_16x16x32_bf16: lane l has row (column) l % 16, K 8 (l / 16) .. + 7.
  // K-contiguous: chunk 4 t + l / 16 of its row, t the K32 step. K-major: two transposing reads (K rows +0
  // and +4), lane l addressing the 8-byte piece l % 4 of K row 32 t + 8 (l / 16) + l / 4 % 4; the swizzle
  // puts the 8 K rows and 2 chunks that 32 lanes read on 16 bank groups.
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(smem));
  const int kr = 8 * (lane >> 4) + ((lane >> 2) & 3);
  const uint32_t vc = (lane & 15) * 128 + (((lane >> 4) ^ ((lane >> 1) & 7)) << 4);  // step 1: chunk ^ 4
  const uint32_t base_a = lds0 + (kAK ? vc + wm * kMB * 32 * 128 : kr * (kTM * 2) + (lane & 1) * 8);
  const uint32_t base_b = lds0 + (kBK ? vc + wn * kNB * 32 * 128 : kr * (kTN * 2) + (lane & 1) * 8);
  const int ksa = k_swizzle<kTM>(kr), ksb = k_swizzle<kTN>(kr), kc = (lane >> 1) & 1;
#define TM_RD(dst, base, imm) asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(dst) : "v"(base), "i"(imm))
#define TM_TR(dst, base, imm) asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(dst) : "v"(base), "i"(imm))
  bf16x8 a8[2][kAK ? kMB : 1], b8[2][kBK ? kFB : 1];
  bf16x4 a4[2][kAK ? 1 : 2 * kMB], b4[2][kBK ? 1 : 2 * kFB];
  auto rd_a = [&](int t, int h, uint32_t ua, int i) {  // read i of step t, half h, from the unit at ua
    if constexpr (kAK) TM_RD(a8[h][i], (base_a ^ (t * 64)) + ua, (h * kMB + i) * 16 * 128);
    else
      TM_TR(a4[h][i], base_a + ua + ((2 * (wm * 2 * kMB + h * kMB + (i >> 1)) + kc) ^ ksa) * 16,
            t * 64 * kTM + (i & 1) * 4 * kTM * 2);
  };
  auto rd_b = [&](int t, uint32_t ub, int i) {
    if constexpr (kBK) TM_RD(b8[t][i], (base_b ^ (t * 64)) + ub, i * 16 * 128);
    else
      TM_TR(b4[t][i], base_b + ub + ((2 * (wn * kFB + (i >> 1)) + kc) ^ ksb) * 16,
            t * 64 * kTN + (i & 1) * 4 * kTN * 2);
  };
  // waits for the reads of A's half h and (t >= 0) of B's step t; naming every fragment keeps the MFMAs that
  // use them behind the wait
  auto wait = [&](int h, int t) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int i = 0; i < kRdA; ++i) {
      if constexpr (kAK) asm volatile("" : "+v"(a8[h][i]));
      else asm volatile("" : "+v"(a4[h][i]));
    }
    if (t >= 0)
#pragma unroll
      for (int i = 0; i < kRdB; ++i) {
        if constexpr (kBK) asm volatile("" : "+v"(b8[t][i]));
        else asm volatile("" : "+v"(b4[t][i]));
      }
  };
  auto afrag = [&](int h, int i) {
    if constexpr (kAK) return a8[h][i];
    else return __builtin_shufflevector(a4[h][2 * i], a4[h][2 * i + 1], 0, 1, 2, 3, 4, 5, 6, 7);
  };
  auto bfrag = [&](int t, int i) {
    if constexpr (kBK) return b8[t][i];
    else return __builtin_shufflevector(b4[t][2 * i], b4[t][2 * i + 1], 0, 1, 2, 3, 4, 5, 6, 7);
  };

  // ---- five units of LDS in a ring: A 0, B 0, A 1, B 1, A 2, ...
  auto after = [&](uint32_t u, int n) {  // the unit n on
    u += n * kUnit;
    return u >= static_cast<uint32_t>(C::kLds) ? u - C::kLds : u;
  };
  uint8_t* const mine = smem + wave * 1024;
  Feed<kTM, kAK, true, kPairs, kRagged, kTM, kTN> fa;
  Feed<kTN, kBK, false, kPairs, kRagged, kTM, kTN> fb;
  fa.seek(g, sh, p, lane, wave);
  fb.seek(g, sh, p, lane, wave);
  fa.count(g);
  fb.count(g);
#pragma unroll 1
  for (int i = 0; i < 2; ++i) {
    fa.load_all(g, sh, mine + 2 * i * kUnit, lane, wave);
    fb.load_all(g, sh, mine + (2 * i + 1) * kUnit, lane, wave);
  }
  __builtin_amdgcn_s_waitcnt(waitcnt_vm(fa.kLoads + fb.kLoads));
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  uint32_t ua = 0, free_b = 4 * kUnit;  // the slice's A (its B is in the next unit); the unit of the last slice's B
#pragma unroll
  for (int i = 0; i < kRdA; ++i) rd_a(0, 0, 0, i);
#pragma unroll
  for (int i = 0; i < kRdB; ++i) rd_b(0, kUnit, i);
  wait(0, 0);
  __builtin_amdgcn_sched_barrier(0);

  for (;;) {
    int tile, batch, m0, n0, n_it, it0;
    const int part = part_of(g, sh, p, tile, it0, n_it);
    place<kTM, kTN, kPairs>(g, tile, batch, m0, n0);
    n_it -= it0;
    f32x4 acc[2 * kMB][kFB];
#pragma unroll
    for (int i = 0; i < 2 * kMB; ++i)
#pragma unroll
      for (int j = 0; j < kFB; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    // A slice is four quarters (K32 step t = q / 2, A's half h = q % 2); in each the operands of the next are
    // read, early, so that the products that follow cover them. In the first, A two slices on is loaded
    // into the unit that the last slice's B has left. Before the fourth the workgroup meets: every
    // wave's loads of the next slice have come in, and nobody reads this slice's units any more, so
    // that B two slices on may be loaded into A's.
    for (int it = 0; it < n_it; ++it) {
      const uint32_t ub = after(ua, 1), na = after(ua, 2), nb = after(ua, 3);
      auto quarter = [&](auto which) {
        constexpr int q = decltype(which)::q, t = q / 2, h = q % 2;
        constexpr int kMf = kMB * kFB, kReads = h == 0 ? kRdA : kRdA + kRdB;
        constexpr int kPer = (4 * kReads + 3 * kMf - 1) / (3 * kMf);
        // loads of this quarter, [from, to): A's in three (kRagged: the first), B's in the fourth
        constexpr int from = kRagged || q == 3 ? 0 : fa.kLoads * q / 3;
        constexpr int to = q == 3 ? fb.kLoads : (kRagged ? (q == 0 ? fa.kLoads : 0) : fa.kLoads * (q + 1) / 3);
        bool loads = true;
        if (kRagged && q == 0) {
          loads = fa.plain > 0;
          if (!loads) fa.load_event(g, sh, mine + free_b, lane, wave);
        }
        if (kRagged && q == 3) {
          loads = fb.plain > 0;
          if (!loads) fb.load_event(g, sh, mine + ua, lane, wave);
        }
#pragma unroll
        for (int f = 0; f < kMf; ++f) {  // one MFMA, its share of the reads and of the loads
#pragma unroll
          for (int i = f * kPer; i < (f + 1) * kPer && i < kReads; ++i) {
            if (h == 0) rd_a(t, 1, ua, i);
            else if (i < kRdA) rd_a(t ^ 1, 0, q == 1 ? ua : na, i);
            else rd_b(t ^ 1, q == 1 ? ub : nb, i - kRdA);
          }
          if (to > from && loads)
#pragma unroll
            for (int j = from + f * (to - from) / kMf; j < from + (f + 1) * (to - from) / kMf; ++j) {
              if (q != 3) fa.load(mine + free_b, j);
              else fb.load(mine + ua, j);
            }
          const int jj = f / kFB, ii = f % kFB;
          acc[h * kMB + jj][ii] =
              __builtin_amdgcn_mfma_f32_16x16x32_bf16(bfrag(t, ii), afrag(h, jj), acc[h * kMB + jj][ii], 0, 0, 0);
          __builtin_amdgcn_sched_barrier(0);
        }
        if (kRagged ? q == 0 && loads : q == 2) {
          if (kRagged || fa.plain > 0) fa.next();
          else fa.past_event(g, sh, lane, wave);
        }
        if (q == 3 && loads) {
          if (kRagged || fb.plain > 0) fb.next();
          else fb.past_event(g, sh, lane, wave);
        }
        wait(h ^ 1, h == 1 ? t ^ 1 : -1);
        __builtin_amdgcn_sched_barrier(0);
      };
      quarter(Quarter<0>{});
      quarter(Quarter<1>{});
      quarter(Quarter<2>{});
      __builtin_amdgcn_s_waitcnt(waitcnt_vm(fa.kLoads));
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_sched_barrier(0);
      quarter(Quarter<3>{});
      free_b = ub;
      ua = na;
    }
    if (part >= 0 && g.splits > 1) {
      f32x4* dst = reinterpret_cast<f32x4*>(g.partial) +
                   (partial_at(g, tile, part) * 8 + wave) * (kMB * kNB * 4 * 64) + lane;
#pragma unroll
      for (int jj = 0; jj < 2 * kMB; ++jj)
#pragma unroll
        for (int ii = 0; ii < kFB; ++ii) dst[(jj * kFB + ii) * 64] = acc[jj][ii];
    } else {  // through the unit that B has left
      finish<kMode, C::kHalves, kMB, kNB>(acc, batch, m0 + wm * kMB * 32, n0 + wn * (kPairs ? 32 : 32 * kNB), lane,
                                          lds0 + free_b + wave * C::kStrip);
      __builtin_amdgcn_s_barrier();  // every wave is done with its strip: A's loads follow there
    }
    p += g.wpx;
    if (p >= pend) break;
    // the next tile's first operands again: their registers were the end's
#pragma unroll
    for (int i = 0; i < kRdA; ++i) rd_a(0, 0, ua, i);
#pragma unroll
    for (int i = 0; i < kRdB; ++i) rd_b(0, after(ua, 1), i);
    wait(0, 0);
    __builtin_amdgcn_sched_barrier(0);
  }
  __builtin_amdgcn_s_waitcnt(0);  // the reloads of the last slices
#undef TM_RD
#undef TM_TR
}

// A split tile's parts lie one after the other, each in the order of the accumulators (a wave's 64 lanes of one
// register group consecutive): summed in order, then the end of the tile's.
template <int kMB, int kNB, int kMode>
__global__ __launch_bounds__(256) void lin_finish_kernel(const Args g) {
  using C = Tile<kMB, kNB>;
  __shared__ __attribute__((aligned(1024))) uint8_t strips[4 * C::kStrip];
  const int lane = threadIdx.x & 63;
  const int w4 = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int T = g.tiles_m * g.tiles_n * g.batch, t8 = (T + 7) / 8;
  const int id = static_cast<int>(blockIdx.x) * 4 + w4;  // (split tile, wave, jj)
  const int xcd = id / (8 * kMB) / (t8 - g.whole), t = xcd * t8 + g.whole + id / (8 * kMB) % (t8 - g.whole);
  if (xcd >= 8 || t >= T) return;
  const int wave = (id / kMB) % 8, jj = id % kMB;
  int batch, m0, n0;
  place<C::kTM, C::kTN, kMode == kGate>(g, t, batch, m0, n0);
  constexpr int kVec = kNB * 4;
  const f32x4* src = reinterpret_cast<const f32x4*>(g.partial) +
                     (partial_at(g, t, 0) * 8 + wave) * (kMB * kNB * 4 * 64) + jj * kVec * 64 + lane;
  const int64_t step = 8 * (kMB * kNB * 4 * 64);
  f32x4 sum[kVec];
#pragma unroll
  for (int i = 0; i < kVec; ++i) sum[i] = src[i * 64];
  for (int s = 1; s < g.splits; ++s) {
    const f32x4* from = src + s * step;
    f32x4 v[kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i) v[i] = from[i * 64];
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      sum[i].x += v[i].x;
      sum[i].y += v[i].y;
      sum[i].z += v[i].z;
      sum[i].w += v[i].w;
    }
  }
  f32x4 v[2][2 * kNB];
#pragma unroll
  for (int i = 0; i < kVec; ++i) v[i / (2 * kNB)][i % (2 * kNB)] = sum[i];
  const int wm = wave >> 2, wn = wave & 3;
  finish<kMode, C::kHalves, 1, kNB>(v, batch, m0 + (wm * kMB + jj) * 32, n0 + wn * (kMode == kGate ? 32 : 32 * kNB), lane,
                            static_cast<uint32_t>(reinterpret_cast<uintptr_t>(strips)) + w4 * C::kStrip);
}

// ------------------------------------------------------------------------------ few rows
//
// The forward products of up to 16 kMT rows (a token, a short sequence's end): bound by the weight's bytes, or,
// where those are few, by the latency of one launch. A workgroup takes 32 output columns (with a gate 32 of
// each weight), kNarrow 16, which puts twice as many CUs to work; its waves take 64 K each in turn and keep
// the whole result, which they add up in LDS in order. An operand's 64 K of a row are 128 bytes of four
// lanes, 32 each: the two MFMAs of a step take the lanes' first and second 16 bytes, the same K of both
// operands. Nothing is loaded twice, so nothing goes through LDS on the way in. The end is the tiles'.
// (Microseconds with 16 columns / 32: 1 x 1024 -> 2816 3.9 / 5.1, 1 x 2816 -> 1024 6.1 / 8.7, 1 x 9728 -> 2560
// 14.2 / 22.8, the gate of 1 x 2560 -> 9728 20.4 / 28.4, 4.9 TB/s.)
template <int kMT, int kMode, bool kNarrow = false>
struct Few {
  // few registers a wave in 16 waves: kLinear's end takes over 128, kNarrow loads more steps at a time
  static constexpr int kWaves = kNarrow || kMT == 4 || kMode == kLinear ? 8 : 16;
  static constexpr int kCols = kNarrow ? 16 : 32;
  static constexpr int kLds = kWaves * kMT * (kCols / 16 * (kMode == kGate ? 2 : 1)) * 1024 + 8192;
};

template <int kMT, int kMode, bool kNarrow>
__global__ __launch_bounds__((Few<kMT, kMode, kNarrow>::kWaves * 64)) void lin_rows_kernel(const Args g) {
  using F = Few<kMT, kMode, kNarrow>;
  constexpr bool kPairs = kMode == kGate;
  constexpr int kFrags = F::kCols / 16, kNT = kPairs ? 2 * kFrags : kFrags, kWaves = F::kWaves, kSums = (kMT + 1) / 2;
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = static_cast<int>(blockIdx.x) * F::kCols, r = lane & 15, c = lane >> 4;
  const char *pw[kNT], *px[kMT];
#pragma unroll
  for (int t = 0; t < kNT; ++t)
    pw[t] = (t >= kFrags ? g.b1 : g.b0) + min(n0 + 16 * (t % kFrags) + r, g.n - 1) * g.b_ld + c * 32;
#pragma unroll
  for (int t = 0; t < kMT; ++t) px[t] = g.a + min(16 * t + r, g.m - 1) * g.a_ld + c * 32;
  f32x4 acc[kMT][kNT];
#pragma unroll
  for (int i = 0; i < kMT; ++i)
#pragma unroll
    for (int j = 0; j < kNT; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  // several steps' loads at a time in flight
  constexpr int kWide = kMT == 4 ? 1 : (kMT == 2 ? 2 : 4) / (kPairs ? 2 : 1);
  constexpr int kBatch = !kNarrow ? kWide : kMT == 4 ? 2 : kMT == 2 ? (kPairs ? 2 : 4) : (kPairs ? 4 : 6), kStep = kWaves * kSliceK;
  for (int k0 = wave * kSliceK; k0 < g.ka; k0 += kBatch * kStep) {
    bf16x8 w[kBatch][kNT][2], x[kBatch][kMT][2];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int k = k0 + b * kStep;
      if (k >= g.ka) break;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const bool in = k + c * 16 + u * 8 < g.ka;
#pragma unroll
        for (int t = 0; t < kNT; ++t) {
          w[b][t][u] = bf16x8{};
          if (in) w[b][t][u] = *reinterpret_cast<const bf16x8*>(pw[t] + static_cast<int64_t>(k) * 2 + u * 16);
        }
#pragma unroll
        for (int t = 0; t < kMT; ++t) {
          x[b][t][u] = bf16x8{};
          if (in) x[b][t][u] = *reinterpret_cast<const bf16x8*>(px[t] + static_cast<int64_t>(k) * 2 + u * 16);
        }
      }
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      if (k0 + b * kStep >= g.ka) break;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < kMT; ++i)
#pragma unroll
          for (int j = 0; j < kNT; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[b][j][u], x[b][i][u], acc[i][j], 0, 0, 0);
    }
  }
  f32x4* part = reinterpret_cast<f32x4*>(smem);
#pragma unroll
  for (int i = 0; i < kMT; ++i)
#pragma unroll
    for (int j = 0; j < kNT; ++j) part[((wave * kMT + i) * kNT + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  if (wave >= kSums) return;
  f32x4 sum[2][kPairs ? 4 : 2] = {};
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int j = 0; j < kNT; ++j) {
      if (2 * wave + h >= kMT) continue;
      f32x4& to = sum[h][j / kFrags * 2 + j % kFrags];
#pragma unroll
      for (int w = 0; w < kWaves; ++w) to += part[((w * kMT + 2 * wave + h) * kNT + j) * 64 + lane];
    }
  finish<kMode, false, 1, kPairs ? 2 : 1, kNarrow>(sum, 0, wave * 32, n0, lane,
                                                   static_cast<uint32_t>(reinterpret_cast<uintptr_t>(smem)) +
                                                       kWaves * kMT * kNT * 1024 + wave * 4096);
}

// ------------------------------------------------------------------------------ the host's side

constexpr int64_t kPad = 64;  // [d0 | d1]: each half is padded to a multiple of this
constexpr int64_t kMaxPartialBytes = int64_t(2) << 30;
// Measured on MI355X: microseconds of a slice and of a tile's end, by tile, fitted to a sweep of 15 tilings and
// splits of 22 products (the block's forward, gradient and weight-gradient products at 8192 rows and some of
// 1999 rows), before the ends got their present form: of 8192 x 9728 -> 2560's 320 tiles of 256 x 256, 256 whole and the
// others in four parts took 366 us then, 417 unsplit, 390 in tiles of 192 x 256. The choice takes at most 2-3%
// more time than the best of the 15, then and on 28 products with the present ends. The ends of a round of tiles come together and are bound by memory: the gate's, by
// what they read and write more.
struct Cost {
  int mb, nb;
  double slice, end;
};
constexpr Cost kCosts[] = {{4, 2, 1.25, 7.0}, {3, 2, 1.24, 3.8}, {2, 2, 0.95, 4.0}, {2, 1, 1.0, 2.9}};
constexpr double kUsSliceAlone = 0.62, kUsEndAlone = 3.3;  // 128 x 128 tiles, one workgroup on a CU instead of two
constexpr double kUsLaunch = 3.0, kUsReduce = 3.8, kBytesPerUs = 5.7e6;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// What a call computes, in the kernel's terms.
struct Product {
  int64_t m, n, slices, batch;
  bool gate;    // n counts features, a tile has half as many as columns
  double ends;  // what a tile's end moves, to a plain one's
};

struct Plan {
  int mb, nb;      // tile of 64 mb x 128 nb
  int64_t whole;   // an XCD's tiles before its split ones
  int64_t splits;  // of those
  double us;
};

int64_t tiles_of(const Product& q, int mb, int nb) {
  return ceil_div(q.m, 64 * mb) * ceil_div(q.n, 128 * nb / (q.gate ? 2 : 1)) * q.batch;
}

// Split tiles' parts in the workspace.
int64_t parts_of(const Product& q, int mb, int nb, int64_t whole, int64_t splits) {
  return splits > 1 ? 8 * (ceil_div(tiles_of(q, mb, nb), 8) - whole) * splits : 0;
}

Plan plan_of(const Product& q, const Cost& c, int64_t whole, int64_t splits) {
  const int64_t per_xcd = ceil_div(tiles_of(q, c.mb, c.nb), 8), rest = (per_xcd - whole) * splits;
  const int64_t per = ceil_div(q.slices, splits), parts = parts_of(q, c.mb, c.nb, whole, splits);
  const bool pair = c.mb * c.nb == 2;
  double us = kUsLaunch;
  auto rounds = [&](int64_t n, int64_t slices, bool ends) {
    const double end = ends ? c.end * q.ends : c.end;
    if (!pair) return ceil_div(n, 32) * (slices * c.slice + end);
    if (whole == 0 && n <= 32) return slices * kUsSliceAlone + kUsEndAlone * (ends ? q.ends : 1.0);
    return ceil_div(n, 64) * (slices * c.slice + end);
  };
  us += rounds(whole, q.slices, true) * (whole > 0) + rounds(rest, per, splits == 1) * (rest > 0);
  if (parts)  // written, read and added up, and the split tiles' ends
    us += kUsReduce + static_cast<double>(parts) * (64 * c.mb * 128 * c.nb) *
                          (8.0 + 2.0 * (q.ends - 1.0) / static_cast<double>(splits)) / kBytesPerUs;
  return {c.mb, c.nb, whole, splits, us};
}

// The tile, which of the tiles are split, and in how many parts, with the least estimated time: none, all, or
// those that whole rounds over the CUs leave over.
Plan best_plan(const Product& q) {
  Plan best = {0, 0, 0, 0, 0.0};
  for (const Cost& c : kCosts) {
    if (c.mb == 2 && (c.nb == 2) != q.gate) continue;
    const int64_t per_xcd = ceil_div(tiles_of(q, c.mb, c.nb), 8), room = c.mb * c.nb == 2 ? 64 : 32;
    const int64_t full = per_xcd / room * room;
    for (int64_t s = 1; s <= 64 && s <= q.slices; ++s) {
      if (ceil_div(q.slices, ceil_div(q.slices, s)) != s) continue;  // some part would be empty
      for (int64_t whole : {int64_t(0), full}) {
        if ((s == 1 && whole) || whole == per_xcd) continue;
        if (parts_of(q, c.mb, c.nb, whole, s) * (64 * c.mb) * (128 * c.nb) * 4 > kMaxPartialBytes) continue;
        const Plan p = plan_of(q, c, whole, s);
        if (best.splits == 0 || p.us < best.us) best = p;
        if (full == 0) break;
      }
    }
  }
  return best;
}

size_t partial_bytes(const Product& q, const Plan& p) {
  return static_cast<size_t>(parts_of(q, p.mb, p.nb, p.whole, p.splits)) * (64 * p.mb) * (128 * p.nb) * sizeof(float);
}

Product product_of(int op, int64_t rows, int64_t inp, int64_t out, bool two) {
  switch (op) {
    case TM_LIN_FORWARD: return {rows, out, ceil_div(inp, kSliceK), 1, false, 1.0};
    case TM_LIN_GATE: return {rows, out, ceil_div(inp, kSliceK), 1, true, 1.85};
    case TM_LIN_GRAD_X: return {rows, inp,
                               two ? 2 * ceil_div(out, kPad) * (kPad / kSliceK) : ceil_div(out, kSliceK), 1,
                               false, 1.0};
    case TM_LIN_GATE_GRAD: return {rows, inp, ceil_div(out, kSliceK), 1, false, 7.5};
    default: return {out, inp, ceil_div(rows, kSliceK), two ? 2 : 1, false, 1.0};
  }
}

// What lin_rows_kernel takes: up to 16 rows, and up to 64 of short K; of somewhat longer K where nothing is held and
// 32 columns to a workgroup do not fill the CUs. (Microseconds against 128 x 128 tiles: 64 x 1024 -> 2816 7.8 / 12.7,
// 32 x 2816 -> 1024 10.6 / 15.0, 64 x 2560 -> 2560 14.4 / 16.6, but 64 x 2816 -> 1024 16.0 / 15.1, 32 x 9728 -> 2560
// 29.9 / 23.3, 32 x 2560 -> 9728 24.3 / 20.4.)
constexpr int64_t kNarrowCols = 8192, kFewElements = 64 * 2560;
bool few_rows(int op, int64_t rows, int64_t inp, int64_t out, bool held) {
  if (op > TM_LIN_GATE || rows > 64) return false;
  return rows <= 16 || inp <= 1536 || (!held && out <= kNarrowCols && rows * inp <= kFewElements);
}

constexpr int kMaxDevices = 64, kKernels = 66;
std::mutex g_mu;
bool g_lds_set[kKernels][kMaxDevices] = {};
int g_cus[kMaxDevices] = {};

// The kernels' dynamic LDS (80-160 KB) exceeds the default limit: raised once per device and kernel,
// with that device current, before the first launch there.
hipError_t allow_lds(hipStream_t stream, int which, const void* fn, int bytes, int* cus) {
  int dev = -1;
  hipError_t e = stream ? hipStreamGetDevice(stream, &dev) : hipGetDevice(&dev);
  if (e != hipSuccess) return e;
  if (dev < 0 || dev >= kMaxDevices) return hipErrorInvalidDevice;
  std::lock_guard<std::mutex> lock(g_mu);
  if (!g_lds_set[which][dev]) {
    int cur = -1;
    e = hipGetDevice(&cur);
    if (e == hipSuccess && cur != dev) e = hipSetDevice(dev);
    if (e == hipSuccess) e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == hipSuccess && g_cus[dev] == 0)
      e = hipDeviceGetAttribute(&g_cus[dev], hipDeviceAttributeMultiprocessorCount, dev);
    if (cur >= 0 && cur != dev) {
      const hipError_t back = hipSetDevice(cur);
      if (e == hipSuccess) e = back;
    }
    if (e != hipSuccess) return e;
    g_lds_set[which][dev] = true;
  }
  *cus = g_cus[dev];
  return hipSuccess;
}

template <int kMB, int kNB, bool kAK, bool kBK, bool kRagged, int kMode>
int launch_one(int which, Args& g, hipStream_t s) {
  using C = Tile<kMB, kNB>;
  int cus = 0;
  const void* fn = reinterpret_cast<const void*>(lin_kernel<kMB, kNB, kAK, kBK, kRagged, kMode>);
  hipError_t e = allow_lds(s, which, fn, C::kLds, &cus);
  if (e != hipSuccess) return lin_fail(TM_ELAUNCH, "tm_lin: LDS attribute: %s", hipGetErrorString(e));
  const int64_t t8 = ceil_div(static_cast<int64_t>(g.tiles_m) * g.tiles_n * g.batch, 8);
  const int64_t per_xcd = g.whole + (t8 - g.whole) * g.splits, room = (cus >= 16 ? cus / 8 : 1) * (2 * C::kLds <= 163840 ? 2 : 1);
  g.wpx = static_cast<int>(per_xcd < room ? per_xcd : room);
  hipLaunchKernelGGL((lin_kernel<kMB, kNB, kAK, kBK, kRagged, kMode>), dim3(static_cast<uint32_t>(8 * g.wpx)), dim3(512), C::kLds,
                     s, g);
  e = hipGetLastError();
  if (e != hipSuccess) return lin_fail(TM_ELAUNCH, "lin_kernel: launch failed: %s", hipGetErrorString(e));
  if (g.splits > 1) {
    const int64_t waves = 8 * (t8 - g.whole) * 8 * kMB;
    hipLaunchKernelGGL((lin_finish_kernel<kMB, kNB, kMode>), dim3(static_cast<uint32_t>(ceil_div(waves, 4))), dim3(256),
                       0, s, g);
    e = hipGetLastError();
    if (e != hipSuccess) return lin_fail(TM_ELAUNCH, "lin_finish_kernel: launch failed: %s", hipGetErrorString(e));
  }
  return TM_OK;
}

// kRagged: some slice reaches past an operand's K.
template <int kMB, int kNB, bool kAK, bool kBK, int kMode>
int launch(int which, Args& g, hipStream_t s) {
  const int seg = g.slices / g.seg;
  if (g.ka == g.slices * kSliceK && g.kb == g.seg * kSliceK && seg * g.seg == g.slices)
    return launch_one<kMB, kNB, kAK, kBK, false, kMode>(2 * which, g, s);
  return launch_one<kMB, kNB, kAK, kBK, true, kMode>(2 * which + 1, g, s);
}

template <int kMT, int kMode, bool kNarrow = false>
int launch_rows(int which, Args& g, hipStream_t s) {
  using F = Few<kMT, kMode, kNarrow>;
  int cus = 0;
  hipError_t e = allow_lds(s, which, reinterpret_cast<const void*>(lin_rows_kernel<kMT, kMode, kNarrow>), F::kLds, &cus);
  if (e != hipSuccess) return lin_fail(TM_ELAUNCH, "tm_lin: LDS attribute: %s", hipGetErrorString(e));
  const int cols = kMode == kGate ? g.n_store : g.n;
  hipLaunchKernelGGL((lin_rows_kernel<kMT, kMode, kNarrow>), dim3(static_cast<uint32_t>(ceil_div(cols, F::kCols))),
                     dim3(F::kWaves * 64), F::kLds, s, g);
  e = hipGetLastError();
  return e == hipSuccess ? TM_OK : lin_fail(TM_ELAUNCH, "lin_rows_kernel: launch failed: %s", hipGetErrorString(e));
}

template <int kMode>
int launch_few(int which, Args& g, hipStream_t s) {
  // 16 columns to a workgroup: not of what is held, whose blocks are 32 x 32, nor where 32 fill the CUs and x
  // is read by each (64 x 1024 -> 9728 16.9 us, 14.6 with 32)
  if (!g.held && (g.m <= 16 || g.n <= kNarrowCols)) {
    if (g.m <= 16) return launch_rows<1, kMode, true>(which + 3, g, s);
    if (g.m <= 32) return launch_rows<2, kMode, true>(which + 4, g, s);
    return launch_rows<4, kMode, true>(which + 5, g, s);
  }
  if constexpr (kMode == kLinear || kMode == kGate)  // what is held
    if (g.m <= 16) return launch_rows<1, kMode>(which, g, s);
  if (g.m <= 32) return launch_rows<2, kMode>(which + 1, g, s);
  return launch_rows<4, kMode>(which + 2, g, s);
}

template <bool kAK, bool kBK, int kMode>
int launch_tile(const Plan& p, int which, Args& g, hipStream_t s) {
  if (p.mb == 4) return launch<4, 2, kAK, kBK, kMode>(3 * which, g, s);
  if (p.mb == 3) return launch<3, 2, kAK, kBK, kMode>(3 * which + 1, g, s);
  return launch<2, kMode == kGate ? 2 : 1, kAK, kBK, kMode>(3 * which + 2, g, s);
}

}  // namespace

extern "C" {

size_t tm_lin_workspace_bytes(int op, int64_t rows, int64_t inp, int64_t out, int two) {
  if (op < TM_LIN_FORWARD || op > TM_LIN_GRAD_W || rows <= 0 || inp <= 0 || out <= 0) return 0;
  if (few_rows(op, rows, inp, out, true)) return 0;  // then also where nothing is held
  const Product q = product_of(op, rows, inp, out, two != 0);
  return partial_bytes(q, best_plan(q));
}

int tm_lin(const tm_lin_t* d, void* d_ws, size_t ws_bytes, void* stream) {
  if (!d) return lin_fail(TM_EINVAL, "tm_lin: null descriptor");
  const int op = d->op;
  if (op < TM_LIN_FORWARD || op > TM_LIN_GRAD_W) return lin_fail(TM_EINVAL, "tm_lin: unknown op %d", op);
  const int64_t kMax = int64_t(1) << 30;
  if (d->rows <= 0 || d->inp <= 0 || d->out <= 0 || d->rows > kMax || d->inp > (1 << 22) || d->out > (1 << 22))
    return lin_fail(TM_EINVAL, "tm_lin: %lld rows, %lld in, %lld out features: each at least 1, at most 2^30, 2^22 and "
                    "2^22", (long long)d->rows, (long long)d->inp, (long long)d->out);
  const bool two = d->b1 != nullptr && op == TM_LIN_GRAD_X, two_out = d->o1 != nullptr && op == TM_LIN_GRAD_W;
  if (!d->a || !d->b0 || !d->o0 || (op == TM_LIN_GATE && !d->b1))
    return lin_fail(TM_EINVAL, "tm_lin: null operand");
  if (!aligned(d->a, 16) || !aligned(d->b0, 16) || !aligned(d->b1, 16) || d->lda % 8 || d->ldb % 8)
    return lin_fail(TM_EINVAL, "tm_lin: operands must be 16-byte aligned, their rows a multiple of 8 elements apart "
                    "(%lld, %lld)", (long long)d->lda, (long long)d->ldb);
  const Product q = product_of(op, d->rows, d->inp, d->out, two || two_out);
  const Plan p = best_plan(q);
  const bool few = few_rows(op, d->rows, d->inp, d->out, d->held != TM_HELD_NOT);
  const size_t need = few ? 0 : partial_bytes(q, p);
  if (need && (!d_ws || ws_bytes < need || !aligned(d_ws, 16)))
    return lin_fail(TM_EINVAL, "tm_lin: workspace of %zu bytes, %zu needed, 16-byte aligned", ws_bytes, need);
  auto up8 = [](int64_t v) { return (v + 7) / 8 * 8; };
  // the stored widths of the operands, and what of K each holds
  const int64_t wide_a = op == TM_LIN_FORWARD || op == TM_LIN_GATE ? up8(d->inp)
                         : op == TM_LIN_GRAD_X && two              ? 2 * ceil_div(d->out, kPad) * kPad
                         : op == TM_LIN_GRAD_W && two_out          ? ceil_div(d->out, kPad) * kPad + up8(d->out)
                                                                   : up8(d->out);
  if (d->lda < wide_a || d->ldb < up8(d->inp) || d->lda >= (1 << 23) || d->ldb >= (1 << 23))
    return lin_fail(TM_EINVAL, "tm_lin: operand rows %lld and %lld elements apart, at least %lld and %lld (whole groups "
                    "of 8) and less than 2^23", (long long)d->lda, (long long)d->ldb, (long long)wide_a,
                    (long long)up8(d->inp));
  Args g = {};
  g.a = reinterpret_cast<const char*>(d->a);
  g.b0 = reinterpret_cast<const char*>(d->b0);
  g.b1 = reinterpret_cast<const char*>(d->b1);
  g.a_ld = d->lda * 2;
  g.b_ld = d->ldb * 2;
  g.m = static_cast<int>(q.m);
  g.n = static_cast<int>(q.n);
  g.slices = g.seg = static_cast<int>(q.slices);
  g.batch = static_cast<int>(q.batch);
  switch (op) {
    case TM_LIN_FORWARD:
    case TM_LIN_GATE:
      g.a_rows = static_cast<int>(d->rows);
      g.b_rows = static_cast<int>(d->out);
      g.ka = g.kb = static_cast<int>(up8(d->inp));
      break;
    case TM_LIN_GRAD_X:
    case TM_LIN_GATE_GRAD:
      g.a_rows = static_cast<int>(d->rows);
      g.b_rows = static_cast<int>(up8(d->inp));
      g.ka = static_cast<int>(wide_a);
      g.kb = static_cast<int>(d->out);
      if (two) g.seg = static_cast<int>(q.slices / 2);
      break;
    default:
      g.a_rows = static_cast<int>(up8(d->out));
      g.b_rows = static_cast<int>(up8(d->inp));
      g.ka = g.kb = static_cast<int>(d->rows);
      g.a_batch = ceil_div(d->out, kPad) * kPad * 2;
  }
  g.whole = static_cast<int>(p.whole);
  g.splits = static_cast<int>(p.splits);
  g.per = static_cast<int>(ceil_div(q.slices, p.splits));
  const int64_t tiles_m = ceil_div(q.m, 64 * p.mb), tiles_n = ceil_div(q.n, 128 * p.nb / (q.gate ? 2 : 1));
  if (tiles_m * tiles_n * q.batch * p.splits > (int64_t(1) << 22))
    return lin_fail(TM_EINVAL, "tm_lin: %lld x %lld x %lld is too large", (long long)d->rows, (long long)d->inp,
                    (long long)d->out);
  g.tiles_m = static_cast<int>(tiles_m);
  g.tiles_n = static_cast<int>(tiles_n);
  g.gm = static_cast<int>(tiles_m < 8 ? tiles_m : 8);
  g.gn = 32 / g.gm;
  g.partial = p.splits > 1 ? static_cast<float*>(d_ws) : nullptr;

  g.o0 = static_cast<char*>(d->o0);
  g.o1 = static_cast<char*>(d->o1);
  g.ldo = d->ldo;
  g.ldo1 = d->ldo1;
  g.out_f32 = d->out_f32 != 0;
  g.act = d->act;
  g.held = d->held;
  g.z0 = static_cast<char*>(d->z0);
  g.z1 = static_cast<char*>(d->z1);
  g.s0 = d->s0;
  g.s1 = d->s1;
  g.ldz = d->ldz;
  const int64_t cols = q.n;
  g.blocks = static_cast<int>(ceil_div(cols, 32));
  g.n_store = g.n;
  if (g.act < 0 || g.act > TM_ACT_GELU_TANH) return lin_fail(TM_EINVAL, "tm_lin: unknown activation %d", d->act);
  if (op != TM_LIN_FORWARD && (d->act || d->bias || d->res))
    return lin_fail(TM_EINVAL, "tm_lin: activation, bias and residual belong to the forward product");
  const bool keeps = op == TM_LIN_FORWARD || op == TM_LIN_GATE, pairs = op == TM_LIN_GATE || op == TM_LIN_GATE_GRAD;
  if (g.held < TM_HELD_NOT || g.held > TM_HELD_E4M3 || (!keeps && !pairs && g.held) ||
      (op == TM_LIN_GATE_GRAD && !g.held))
    return lin_fail(TM_EINVAL, "tm_lin: op %d with held %d", op, d->held);
  if (g.held) {
    if (!d->z0 || (pairs && !d->z1) || !aligned(d->z0, 16) || !aligned(d->z1, 16))
      return lin_fail(TM_EINVAL, "tm_lin: what is held must be 16-byte aligned, not null");
    if (g.held == TM_HELD_BF16 ? d->ldz % 8 || d->ldz < cols || d->ldz - cols >= 8
                               : d->ldz != ceil_div(cols, 32) * 32 || !d->s0 || (pairs && !d->s1))
      return lin_fail(TM_EINVAL, "tm_lin: held rows %lld elements apart for %lld columns: the next multiple of 8 (bf16) "
                      "or of 32, with exponents (e4m3)", (long long)d->ldz, (long long)cols);
  }
  if (pairs) {  // rows of whole vectors that the next product reads
    const int64_t pad = op == TM_LIN_GATE ? up8(cols) : ceil_div(cols, kPad) * kPad;
    g.n_store = static_cast<int>(pad);
    if (g.out_f32 || d->ldo % 8 || d->ldo < (op == TM_LIN_GATE ? pad : 2 * pad) || !aligned(d->o0, 16) ||
        (op == TM_LIN_GATE_GRAD && d->o1 && (d->ldo1 % 8 || d->ldo1 < pad || !aligned(d->o1, 16))))
      return lin_fail(TM_EINVAL, "tm_lin: the gate's outputs are bf16, 16-byte aligned, rows %lld and %lld elements apart "
                      "a multiple of 8 that holds %lld columns each", (long long)d->ldo, (long long)d->ldo1,
                      (long long)pad);
  } else if (d->ldo < cols) {
    return lin_fail(TM_EINVAL, "tm_lin: output rows %lld elements apart for %lld columns", (long long)d->ldo,
                    (long long)cols);
  }
  if (!aligned(d->o0, g.out_f32 ? 4 : 2) || !aligned(d->o1, g.out_f32 ? 4 : 2) || !aligned(d->res, d->res_f32 ? 4 : 2) ||
      !aligned(d->bias, d->bias_f32 ? 4 : 2))
    return lin_fail(TM_EINVAL, "tm_lin: outputs, residual and bias must be aligned to their elements");
  if (d->ldo >= (1 << 24) || d->ldo1 >= (1 << 24) || d->ldr >= (1 << 24) || (d->res && d->ldr < cols) ||
      (two_out && d->ldo1 != d->ldo))  // a lane's offsets have 32 bits
    return lin_fail(TM_EINVAL, "tm_lin: output rows %lld, %lld (the same where a gradient has two outputs) and residual "
                    "rows %lld elements apart, less than 2^24, at least %lld", (long long)d->ldo, (long long)d->ldo1,
                    (long long)d->ldr, (long long)cols);
  g.bias = static_cast<const char*>(d->bias);
  g.bias_f32 = d->bias_f32 != 0;
  g.res = static_cast<const char*>(d->res);
  g.res_f32 = d->res_f32 != 0;
  g.ldr = d->ldr;

  hipStream_t s = static_cast<hipStream_t>(stream);
  if (few) {
    if (op == TM_LIN_GATE) return launch_few<kGate>(kKernels - 24, g, s);
    if (g.bias || g.act || g.held) return launch_few<kLinear>(kKernels - 18, g, s);
    return g.res ? launch_few<kResidual>(kKernels - 12, g, s) : launch_few<kPlain>(kKernels - 6, g, s);
  }
  switch (op) {
    case TM_LIN_FORWARD:
      if (g.bias || g.act || g.held) return launch_tile<true, true, kLinear>(p, 0, g, s);
      return g.res ? launch_tile<true, true, kResidual>(p, 1, g, s) : launch_tile<true, true, kPlain>(p, 2, g, s);
    case TM_LIN_GATE: return launch_tile<true, true, kGate>(p, 3, g, s);
    case TM_LIN_GRAD_X: return launch_tile<true, false, kPlain>(p, 4, g, s);
    case TM_LIN_GATE_GRAD: return launch_tile<true, false, kGateGrad>(p, 5, g, s);
    default: return launch_tile<false, false, kPlain>(p, 6, g, s);
  }
}

}  // extern "C"
