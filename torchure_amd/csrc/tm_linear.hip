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
// One kernel template (lin_kernel) with fp32 accumulation on v_mfma_f32_32x32x16_bf16: 8 wave64, two a
// SIMD, wave (wm, wn) = (w / 4, w % 4) computing 32 kMB x 32 kNB of a 64 kMB x 128 kNB tile. Operands
// stream global -> LDS (global_load_lds, 16 bytes a lane) into two stages of 64-deep K slices. A
// K-contiguous operand lies there in 128-byte rows, chunk c of row r at slot c ^ ((r >> 1) & 7); a
// K-major one in whole rows of the tile's columns, chunk c of row k at slot c ^ (4 (k & 3)), and is
// read transposed (ds_read_b64_tr_b16): in both, the 16 lanes of a read hit 16 bank groups.
//
// Workgroups are persistent. A workgroup's tiles form one stream of K slices: the loads run two
// slices ahead of the products, across tiles, so that a tile starts on operands that came in during
// the one before it; its results leave through a strip of LDS of their own while the next tile's
// loads are in flight. Workgroup w runs on XCD w % 8; each XCD takes a contiguous range of tile
// positions, in groups of gm x gn tiles whose operand panels share its L2.
//
// Edges: rows and columns past an operand's last are loaded again (their results are not stored); K
// past the operand's end is loaded from 16 bytes of zeros, on both sides, so that no garbage meets
// a zero. Products with few tiles are split over K: fp32 partial tiles in the workspace, added in
// split order by lin_finish_kernel, which then does what the unsplit kernel's end does.

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

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

template <typename... A>
int lin_fail(int code, const char* fmt, A... args) {
  return tm_internal_fail(code, fmt, args...);
}

constexpr int kSliceK = 64;  // K depth of one LDS stage

constexpr int waitcnt_vm(int n) { return (n & 15) | ((n >> 4) << 14) | (7 << 4) | (15 << 8); }

__device__ const u32x4 g_zeros = {0, 0, 0, 0};  // what K past an operand's end reads

enum Mode { kLinear, kPlain, kGate, kGateGrad };

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
  int per, splits;          // K slices a position covers
  int tiles_m, tiles_n, batch, gm, gn, wpx;
  // what follows the product
  char* o0;
  char* o1;                 // batch 1's output; gate_grad: silu(g) u
  int64_t ldo, ldo1;        // elements
  int out_f32, out_vec, act;
  int n_store;              // columns of an output row that are written (past n: zeros)
  const char* bias;
  const char* res;
  int64_t ldr;
  int bias_f32, bias_vec, res_f32, res_vec;
  char* z0;                 // pre-activations (gate products), up products
  char* z1;
  uint8_t* s0;              // their block exponents, where they are held as e4m3
  uint8_t* s1;
  int64_t ldz;
  int held, blocks;         // TM_HELD_*; blocks of 32 columns in a row of exponents
  float* partial;
};

// Tile of position p: n-blocks of gn tile columns; inside each, m-blocks of gm tile rows, a
// block's gm x gn tiles consecutive in p.
__device__ __forceinline__ void tile_of(int p, int tiles_m, int tiles_n, int gm, int gn, int& tm, int& tn) {
  const int per_nb = tiles_m * gn;
  const int nb = p / per_nb, rem = p - nb * per_nb;
  const int gn_eff = min(gn, tiles_n - nb * gn);
  const int mb = rem / (gm * gn_eff), rem2 = rem - mb * gm * gn_eff;
  tm = mb * gm + rem2 / gn_eff;
  tn = nb * gn + rem2 % gn_eff;
}

// ------------------------------------------------------------------------------ a tile's results
//
// A wave's accumulators come out in blocks of 32 x 32: register 4 q + e of lane l holds row l % 32, column
// 8 q + 4 (l / 32) + e. Each block goes through this wave's strip of LDS (fp32, 128-byte rows, chunk c of
// row r at slot c ^ ((r >> 1) & 7): a wave's LDS accesses are served in order, so no barrier and no wait
// is needed between its writes and its reads) and is read back in the order of the output's rows: lane l
// has columns 8 (l % 4) .. + 7 of rows l / 4 and 16 + l / 4. From there on every access to memory is 16
// bytes a lane and whole pieces of rows, whatever is fused, and one copy of the code serves all blocks.

typedef const __attribute__((address_space(4))) Args* ArgsPtr;  // the kernel's arguments, where they are

struct Block {
  float v[16];  // [row half][column]
};

// kHalves: a strip of 2 KB, 16 rows at a time (else 4 KB).
template <bool kHalves>
__device__ __forceinline__ void to_rows(Block& b, const f32x16& acc, uint32_t stg, int lane) {
  const int row = lane & 31, sw = (row >> 1) & 7;
#pragma unroll
  for (int h = 0; h < (kHalves ? 2 : 1); ++h) {
    if (!kHalves || (row >> 4) == h) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t at = stg + (kHalves ? row & 15 : row) * 128 + (((2 * q + (lane >> 5)) ^ sw) << 4);
        const f32x4 o = {acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
        asm volatile("ds_write_b128 %0, %1" ::"v"(at), "v"(o) : "memory");
      }
    }
    f32x4 t[4];
    if constexpr (kHalves) {
      const int r = lane >> 2, s = (r >> 1) & 7, c = 2 * (lane & 3);
      asm volatile("ds_read_b128 %0, %2\n\tds_read_b128 %1, %3\n\ts_waitcnt lgkmcnt(0)"
                   : "=&v"(t[0]), "=&v"(t[1])
                   : "v"(stg + r * 128 + ((c ^ s) << 4)), "v"(stg + r * 128 + (((c + 1) ^ s) << 4))
                   : "memory");
    } else {
      const int r = lane >> 2, s = (r >> 1) & 7, c = 2 * (lane & 3);
      const uint32_t a0 = stg + r * 128 + ((c ^ s) << 4), a1 = stg + r * 128 + (((c + 1) ^ s) << 4);
      // 16 rows on: the same slots
      asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %1, %5\n\tds_read_b128 %2, %4 offset:2048\n\t"
                   "ds_read_b128 %3, %5 offset:2048\n\ts_waitcnt lgkmcnt(0)"
                   : "=&v"(t[0]), "=&v"(t[1]), "=&v"(t[2]), "=&v"(t[3])
                   : "v"(a0), "v"(a1)
                   : "memory");
    }
#pragma unroll
    for (int i = 0; i < (kHalves ? 2 : 4); ++i) {
      const int at = (kHalves ? 8 * h : 0) + 4 * i;
      b.v[at] = t[i].x;
      b.v[at + 1] = t[i].y;
      b.v[at + 2] = t[i].z;
      b.v[at + 3] = t[i].w;
    }
  }
}

// Eight bf16 or fp32 values of a row; `left` of them exist, vec: 16-byte pieces.
__device__ __forceinline__ void get8(float (&x)[8], const char* p, bool f32, int left, bool vec) {
  if (vec && left >= 8) {
    if (f32) {
      const f32x4 a = reinterpret_cast<const f32x4*>(p)[0], b = reinterpret_cast<const f32x4*>(p)[1];
      x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
      x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
      const u32x4 a = *reinterpret_cast<const u32x4*>(p);
      x[0] = tm_act::bf16_lo(a.x); x[1] = tm_act::bf16_hi(a.x);
      x[2] = tm_act::bf16_lo(a.y); x[3] = tm_act::bf16_hi(a.y);
      x[4] = tm_act::bf16_lo(a.z); x[5] = tm_act::bf16_hi(a.z);
      x[6] = tm_act::bf16_lo(a.w); x[7] = tm_act::bf16_hi(a.w);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = 0.0f;
      if (e < left)
        x[e] = f32 ? reinterpret_cast<const float*>(p)[e]
                   : __uint_as_float(static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[e]) << 16);
    }
  }
}

__device__ __forceinline__ void put8(char* p, const float* x, bool f32, int left, bool vec) {
  if (f32) {
    if (vec && left >= 8) {
      reinterpret_cast<f32x4*>(p)[0] = f32x4{x[0], x[1], x[2], x[3]};
      reinterpret_cast<f32x4*>(p)[1] = f32x4{x[4], x[5], x[6], x[7]};
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < left) reinterpret_cast<float*>(p)[e] = x[e];
    }
  } else {
    const u32x4 w = {pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7])};
    if (vec && left >= 8) {
      *reinterpret_cast<u32x4*>(p) = w;
    } else {
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < left) reinterpret_cast<uint16_t*>(p)[e] = static_cast<uint16_t>(u[e / 2] >> (16 * (e & 1)));
    }
  }
}

// The largest of a value over the wave's lanes.
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), d)));
  return v;
}

// Where a lane's values of a block are, and which of them exist.
struct Spot {
  int64_t m;        // first row; the second is 16 on
  int n, cols;      // first column; columns left from it
  bool row[2];
};

__device__ __forceinline__ Spot spot_of(ArgsPtr g, int m0, int n0, int lane) {
  Spot s;
  s.m = m0 + (lane >> 2);
  s.n = n0 + 8 * (lane & 3);
  s.cols = g->n - s.n;
  s.row[0] = s.m < g->m;
  s.row[1] = s.m + 16 < g->m;
  return s;
}

__device__ __forceinline__ void mask(Block& b, const Spot& s) {
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (!s.row[i / 8] || i % 8 >= s.cols) b.v[i] = 0.0f;
}

// A block as the backward pass reads it (its values outside the matrix zero): z's padding columns are
// written too.
__device__ __forceinline__ void hold(ArgsPtr g, const Block& b, const Spot& s, int m0, int n0, char* z, uint8_t* exps,
                                     int lane) {
  if (g->held == TM_HELD_BF16) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (s.row[i] && s.n < g->ldz) put8(z + ((s.m + 16 * i) * g->ldz + s.n) * 2, b.v + 8 * i, false, 8, true);
  } else {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) most = max(most, tm_act::finite_bits(b.v[i]));
    const int e = tm_act::block_exponent(wave_max(most));
    const float inv = tm_act::two_to(-e);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float* x = b.v + 8 * i;
      const u32x2 w = {tm_act::encode4(x[0], x[1], x[2], x[3], inv), tm_act::encode4(x[4], x[5], x[6], x[7], inv)};
      if (s.row[i]) *reinterpret_cast<u32x2*>(z + (s.m + 16 * i) * g->ldz + s.n) = w;
    }
    if (lane == 0) exps[static_cast<int64_t>(m0 >> 5) * g->blocks + (n0 >> 5)] = static_cast<uint8_t>(e + 127);
  }
}

__device__ __forceinline__ void held_block(ArgsPtr g, Block& b, const Spot& s, int m0, int n0, const char* z,
                                           const uint8_t* exps) {
  if (g->held == TM_HELD_BF16) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float x[8] = {};
      if (s.row[i] && s.n < g->ldz) get8(x, z + ((s.m + 16 * i) * g->ldz + s.n) * 2, false, 8, true);
#pragma unroll
      for (int e = 0; e < 8; ++e) b.v[8 * i + e] = x[e];
    }
  } else {
    const float scale =
        tm_act::two_to(static_cast<int>(exps[static_cast<int64_t>(m0 >> 5) * g->blocks + (n0 >> 5)]) - 127);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      u32x2 w = {0, 0};
      if (s.row[i]) w = *reinterpret_cast<const u32x2*>(z + (s.m + 16 * i) * g->ldz + s.n);
      const f32x4 lo = tm_act::decode4(w.x, scale), hi = tm_act::decode4(w.y, scale);
      float* x = b.v + 8 * i;
      x[0] = lo.x; x[1] = lo.y; x[2] = lo.z; x[3] = lo.w;
      x[4] = hi.x; x[5] = hi.y; x[6] = hi.z; x[7] = hi.w;
    }
  }
}

// y = act(z + b) + r, and z as it is kept. The products' fp32 sums are rounded once, in y's type; z
// is rounded to what the backward pass reads.
__device__ __forceinline__ void end_linear(ArgsPtr g, Block& b, int m0, int n0, int lane) {
  if (m0 >= g->m || n0 >= g->n) return;
  const Spot s = spot_of(g, m0, n0, lane);
  if (g->bias) {
    float x[8];
    get8(x, g->bias + static_cast<int64_t>(s.n) * (g->bias_f32 ? 4 : 2), g->bias_f32, s.cols, g->bias_vec);
#pragma unroll
    for (int i = 0; i < 16; ++i) b.v[i] += x[i % 8];
  }
  if (g->held) {
    if (m0 + 32 > g->m || n0 + 32 > g->n) mask(b, s);
    hold(g, b, s, m0, n0, g->z0, g->s0, lane);
  }
  const int act = g->act;
  auto each = [&](auto f) {
#pragma unroll
    for (int i = 0; i < 16; ++i) b.v[i] = f(b.v[i]);
  };
  if (act == tm_act::kRelu) each([](float z) { return tm_act::act1(tm_act::kRelu, z); });
  else if (act == tm_act::kSilu) each([](float z) { return tm_act::act1(tm_act::kSilu, z); });
  else if (act == tm_act::kGelu) each([](float z) { return tm_act::act1(tm_act::kGelu, z); });
  else if (act == tm_act::kGeluTanh) each([](float z) { return tm_act::act1(tm_act::kGeluTanh, z); });
  const int size_r = g->res_f32 ? 4 : 2, size_o = g->out_f32 ? 4 : 2;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (!s.row[i] || s.cols <= 0) continue;
    if (g->res) {
      float x[8];
      get8(x, g->res + ((s.m + 16 * i) * g->ldr + s.n) * size_r, g->res_f32, s.cols, g->res_vec);
#pragma unroll
      for (int e = 0; e < 8; ++e) b.v[8 * i + e] += x[e];
    }
    put8(g->o0 + ((s.m + 16 * i) * g->ldo + s.n) * size_o, b.v + 8 * i, g->out_f32, s.cols, g->out_vec);
  }
}

__device__ __forceinline__ void end_plain(ArgsPtr g, int batch, Block& b, int m0, int n0, int lane) {
  if (m0 >= g->m || n0 >= g->n) return;
  const Spot s = spot_of(g, m0, n0, lane);
  const int size_o = g->out_f32 ? 4 : 2;
  char* out = batch ? g->o1 : g->o0;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (s.row[i] && s.cols > 0)
      put8(out + ((s.m + 16 * i) * g->ldo + s.n) * size_o, b.v + 8 * i, g->out_f32, s.cols, g->out_vec);
}

// h = silu(g) u of 32 features, g and u kept on the way. Columns of padding are zeros.
__device__ __forceinline__ void end_gate(ArgsPtr g, Block& gate, Block& up, int m0, int n0, int lane) {
  if (m0 >= g->m || n0 >= g->n_store) return;
  const Spot s = spot_of(g, m0, n0, lane);
  if (m0 + 32 > g->m || n0 + 32 > g->n) {
    mask(gate, s);
    mask(up, s);
  }
  if (g->held && n0 < g->n) {
    hold(g, gate, s, m0, n0, g->z0, g->s0, lane);
    hold(g, up, s, m0, n0, g->z1, g->s1, lane);
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) gate.v[i] = gate.v[i] * tm_act::sigmoid(gate.v[i]) * up.v[i];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (s.row[i] && s.n < g->n_store)
      put8(g->o0 + ((s.m + 16 * i) * g->ldo + s.n) * 2, gate.v + 8 * i, false, 8, true);
}

// From dh: d_gate and d_up (columns 0.. and n_store.. of o0's rows) and silu(g) u (o1), g and u as held.
__device__ __forceinline__ void end_gate_grad(ArgsPtr g, Block& d, int m0, int n0, int lane) {
  if (m0 >= g->m || n0 >= g->n_store) return;
  const Spot s = spot_of(g, m0, n0, lane);
  Block gate = {}, up = {};
  if (n0 < g->n) {
    held_block(g, gate, s, m0, n0, g->z0, g->s0);
    held_block(g, up, s, m0, n0, g->z1, g->s1);
  }
  if (n0 + 32 > g->n) mask(d, s);  // g and u are zero there
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float z = gate.v[i], q = tm_act::sigmoid(z), a = z * q;
    gate.v[i] = d.v[i] * up.v[i] * tm_act::silu_grad(z, q);
    d.v[i] *= a;
    up.v[i] *= a;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (!s.row[i] || s.n >= g->n_store) continue;
    char* o = g->o0 + ((s.m + 16 * i) * g->ldo + s.n) * 2;
    put8(o, gate.v + 8 * i, false, 8, true);
    put8(o + static_cast<int64_t>(g->n_store) * 2, d.v + 8 * i, false, 8, true);
    if (g->o1) put8(g->o1 + ((s.m + 16 * i) * g->ldo1 + s.n) * 2, up.v + 8 * i, false, 8, true);
  }
}

// The blocks acc(0) .. acc(kBlocks - 1) of a wave, block b at row m(b), column n(b). One copy of the ends: a
// loop over the blocks whose first step picks the block's registers.
template <int kMode, bool kHalves, int kNB, int kMBs>
__device__ __forceinline__ void finish(f32x16 (&acc)[kMBs][kNB], int batch, int m0, int n0, int lane, uint32_t stg) {
  ArgsPtr g = (ArgsPtr)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(g));  // read again for each tile: held in registers through the product they spill
  constexpr int kPer = kMode == kGate ? 2 : 1;
#pragma unroll 1
  for (int b = 0; b < kMBs * kNB / kPer; ++b) {
    Block x, y;
#pragma unroll
    for (int c = 0; c < kMBs * kNB / kPer; ++c)
      if (b == c) {
        to_rows<kHalves>(x, acc[c * kPer / kNB][c * kPer % kNB], stg, lane);
        if constexpr (kMode == kGate) to_rows<kHalves>(y, acc[c * kPer / kNB][c * kPer % kNB + 1], stg, lane);
      }
    const int m = m0 + b * kPer / kNB * 32, n = n0 + (kMode == kGate ? 0 : b % kNB * 32);
    if constexpr (kMode == kLinear) end_linear(g, x, m, n, lane);
    else if constexpr (kMode == kPlain) end_plain(g, batch, x, m, n, lane);
    else if constexpr (kMode == kGate) end_gate(g, x, y, m, n, lane);
    else end_gate_grad(g, x, m, n, lane);
  }
}

// ------------------------------------------------------------------------------ the product

template <int kMB, int kNB>
struct Tile {
  static constexpr int kTM = 64 * kMB, kTN = 128 * kNB, kStage = (kTM + kTN) * 128;
  static constexpr bool kHalves = kMB * kNB == 2;         // 80 KB: two workgroups a CU
  static constexpr int kStrip = kHalves ? 2048 : 4096;  // one wave's
  static constexpr int kLds = 2 * kStage + 8 * kStrip;
};

// Position -> split, batch and the tile's first row and column (gate: feature).
template <int kTM, int kTN, bool kHalf>
__device__ __forceinline__ void place(const Args& g, int p, int& split, int& batch, int& m0, int& n0) {
  const int tb = g.tiles_m * g.tiles_n, t_all = tb * g.batch;
  split = p / t_all;
  const int t = p - split * t_all;
  batch = t / tb;
  int tm, tn;
  tile_of(t - batch * tb, g.tiles_m, g.tiles_n, g.gm, g.gn, tm, tn);
  m0 = tm * kTM;
  n0 = tn * (kHalf ? kTN / 2 : kTN);
}

template <int kMB, int kNB, bool kAK, bool kBK, int kMode>
__global__ __launch_bounds__(512, kMB * kNB == 2 ? 4 : 2) void lin_kernel(const Args g) {
  using C = Tile<kMB, kNB>;
  constexpr int kTM = C::kTM, kTN = C::kTN, kStage = C::kStage;
  constexpr int kLoads = (kTM + kTN) / 64, kInA = kTM / 8, kInB = kTN / 8;
  constexpr int kRdA = kAK ? kMB : 2 * kMB, kRdB = kBK ? kNB : 2 * kNB, kRd = kRdA + kRdB, kMf = kMB * kNB;
  constexpr bool kPairs = kMode == kGate;
  static_assert(!kPairs || (kNB == 2 && kBK), "gate and up columns alternate by 32 within a wave");
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const int P = g.tiles_m * g.tiles_n * g.batch * g.splits;
  const int p8 = (P + 7) / 8;
  const int pend = min((static_cast<int>(blockIdx.x % 8) + 1) * p8, P);
  int p = static_cast<int>(blockIdx.x % 8) * p8 + static_cast<int>(blockIdx.x / 8);
  if (p >= pend) return;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 2, wn = wave & 3;

  // ---- the loader's place: position lp, slice lit of lend, operand pointers at that slice
  int lp = p, lit = 0, lend = 0;
  const char *la = nullptr, *lb = nullptr, *lb2 = nullptr;
  uint32_t off[kLoads];  // this lane's bytes past the operand's pointer, load j
  const int64_t step_a = kAK ? kSliceK * 2 : kSliceK * g.a_ld, step_b = kBK ? kSliceK * 2 : kSliceK * g.b_ld;
  int64_t col_b = 0;
  // Load q = kLoads wave + j: 1 KB of A's stage (q < kInA), then of B's. K-contiguous: 8 rows;
  // K-major: whole K rows of the tile's columns.
  auto k_contig = [&](int qq, int& r, int& c) {
    r = qq * 8 + lane / 8;
    c = (lane % 8) ^ ((r >> 1) & 7);
  };
  auto k_major = [&](int qq, int cpr, int& kr, int& c) {
    kr = qq * (64 / cpr) + lane / cpr;
    c = (lane % cpr) ^ (4 * (kr & 3));
  };
  auto seek = [&](int pos) {
    int split, batch, m0, n0;
    place<kTM, kTN, kPairs>(g, pos, split, batch, m0, n0);
    lit = split * g.per;
    lend = min(lit + g.per, g.slices);
    if constexpr (kAK) la = g.a + m0 * g.a_ld + static_cast<int64_t>(lit) * (kSliceK * 2);
    else la = g.a + batch * g.a_batch + static_cast<int64_t>(m0) * 2 + lit * step_a;
    if constexpr (kBK) {
      const int64_t at = n0 * g.b_ld + static_cast<int64_t>(lit) * (kSliceK * 2);
      lb = g.b0 + at;
      if constexpr (kPairs) lb2 = g.b1 + at;
    } else {
      col_b = static_cast<int64_t>(n0) * 2;
      lb = lit >= g.seg ? g.b1 + col_b + (lit - g.seg) * step_b : g.b0 + col_b + lit * step_b;
    }
    const int left_a = g.a_rows - m0, left_b = g.b_rows - n0;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int q = wave * kLoads + j;
      int r, c;
      if (q < kInA) {
        if constexpr (kAK) {
          k_contig(q, r, c);
          off[j] = static_cast<uint32_t>(min(r, left_a - 1)) * static_cast<uint32_t>(g.a_ld) + c * 16;
        } else {
          k_major(q, kTM / 8, r, c);
          off[j] = static_cast<uint32_t>(r) * static_cast<uint32_t>(g.a_ld) + min(8 * c, left_a - 8) * 2;
        }
      } else {
        if constexpr (kBK) {
          k_contig(q - kInA, r, c);
          const int row = kPairs ? (r >> 6) * 32 + (r & 31) : r;
          off[j] = static_cast<uint32_t>(min(row, left_b - 1)) * static_cast<uint32_t>(g.b_ld) + c * 16;
        } else {
          k_major(q - kInA, kTN / 8, r, c);
          off[j] = static_cast<uint32_t>(r) * static_cast<uint32_t>(g.b_ld) + min(8 * c, left_b - 8) * 2;
        }
      }
    }
  };
  auto advance = [&]() {
    if (lit + 1 < lend) {
      ++lit;
      la += step_a;
      if (!kBK && lit == g.seg) lb = g.b1 + col_b;
      else lb += step_b;
      if (kPairs) lb2 += step_b;
    } else if (lp + g.wpx < pend) {
      lp += g.wpx;
      seek(lp);
    }  // else: the last slice again, which nothing reads
  };
  auto to_lds = [&](const char* from, int stage, int q) {
    __builtin_amdgcn_global_load_lds((const void __attribute__((address_space(1)))*)from,
                                     (void __attribute__((address_space(3)))*)(smem + stage * kStage + q * 1024), 16, 0, 0);
  };
  auto source = [&](int j) {
    const int q = wave * kLoads + j;
    if (q < kInA) return la + off[j];
    if (kPairs && (((q - kInA) >> 2) & 1)) return lb2 + off[j];
    return lb + off[j];
  };
  auto load = [&](int stage, int j) { to_lds(source(j), stage, wave * kLoads + j); };
  // whether the loader's slice reaches past an operand's K; its loads then
  auto ragged = [&]() {
    const int kb0 = !kBK && lit >= g.seg ? lit - g.seg : lit;
    return (lit + 1) * kSliceK > g.ka || (kb0 + 1) * kSliceK > g.kb;
  };
  auto load_ragged = [&](int stage) {
    const int kb0 = !kBK && lit >= g.seg ? lit - g.seg : lit;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int q = wave * kLoads + j;
      int r, c;
      bool in;
      if (q < kInA) {
        if constexpr (kAK) {
          k_contig(q, r, c);
          in = lit * kSliceK + c * 8 < g.ka;
        } else {
          k_major(q, kTM / 8, r, c);
          in = lit * kSliceK + r < g.ka;
        }
      } else {
        if constexpr (kBK) {
          k_contig(q - kInA, r, c);
          in = lit * kSliceK + c * 8 < g.kb;
        } else {
          k_major(q - kInA, kTN / 8, r, c);
          in = kb0 * kSliceK + r < g.kb;
        }
      }
      to_lds(in ? source(j) : reinterpret_cast<const char*>(&g_zeros), stage, q);
    }
  };

  // ---- fragments: K-contiguous, row lane % 32 of a block, chunk 2 kk + lane / 32; K-major, two
  // transposing reads (K rows +0 and +4) of 8-byte pieces
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(smem));
  const int tx = (lane >> 5) ^ ((lane >> 1) & 7);
  uint32_t vk[4];
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) vk[kk] = lds0 + (lane & 31) * 128 + (((2 * kk) ^ tx) * 16);
  const int s16 = lane & 15, s4 = s16 >> 2;
  const int lcf = ((lane >> 4) & 1) * 2 + ((s16 & 3) >> 1);
  uint32_t ba[kMB], bb[kNB];
#pragma unroll
  for (int i = 0; i < kMB; ++i)
    ba[i] = lds0 + (8 * (lane >> 5) + s4) * (kTM * 2) + (s16 & 1) * 8 + (4 * ((wm * kMB + i) ^ s4) + lcf) * 16;
#pragma unroll
  for (int i = 0; i < kNB; ++i)
    bb[i] = lds0 + kInA * 1024 + (8 * (lane >> 5) + s4) * (kTN * 2) + (s16 & 1) * 8 +
            (4 * ((wn * kNB + i) ^ s4) + lcf) * 16;
  const uint32_t off_a = wm * kMB * 32 * 128, off_b = kInA * 1024 + wn * kNB * 32 * 128;
#define TM_RD(dst, base, imm) asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(dst) : "v"(base), "i"(imm))
#define TM_TR(dst, base, imm) asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(dst) : "v"(base), "i"(imm))
  bf16x8 a8[2][kAK ? kMB : 1], b8[2][kBK ? kNB : 1];
  bf16x4 a4[2][kAK ? 1 : 2 * kMB], b4[2][kBK ? 1 : 2 * kNB];
  auto rd = [&](int z, uint32_t so, int kk, int i) {
    if (i < kRdA) {
      if constexpr (kAK) TM_RD(a8[z][i], vk[kk] + so + off_a, i * 32 * 128);
      else TM_TR(a4[z][i], ba[i >> 1] + so, kk * 16 * kTM * 2 + (i & 1) * 4 * kTM * 2);
    } else {
      const int h = i - kRdA;
      if constexpr (kBK) TM_RD(b8[z][h], vk[kk] + so + off_b, h * 32 * 128);
      else TM_TR(b4[z][h], bb[h >> 1] + so, kk * 16 * kTN * 2 + (h & 1) * 4 * kTN * 2);
    }
  };
  // waits for set z's reads; naming every fragment keeps the MFMAs that use them behind the wait
  auto wait = [&](int z) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int i = 0; i < kRdA; ++i) {
      if constexpr (kAK) asm volatile("" : "+v"(a8[z][i]));
      else asm volatile("" : "+v"(a4[z][i]));
    }
#pragma unroll
    for (int i = 0; i < kRdB; ++i) {
      if constexpr (kBK) asm volatile("" : "+v"(b8[z][i]));
      else asm volatile("" : "+v"(b4[z][i]));
    }
  };
  auto afrag = [&](int z, int i) {
    if constexpr (kAK) return a8[z][i];
    else return __builtin_shufflevector(a4[z][2 * i], a4[z][2 * i + 1], 0, 1, 2, 3, 4, 5, 6, 7);
  };
  auto bfrag = [&](int z, int i) {
    if constexpr (kBK) return b8[z][i];
    else return __builtin_shufflevector(b4[z][2 * i], b4[z][2 * i + 1], 0, 1, 2, 3, 4, 5, 6, 7);
  };
  auto load_slice = [&](int stage) {
    if (ragged()) {
      load_ragged(stage);
    } else {
#pragma unroll
      for (int j = 0; j < kLoads; ++j) load(stage, j);
    }
    advance();
  };

  seek(p);
  load_slice(0);
  load_slice(1);
  __builtin_amdgcn_s_waitcnt(waitcnt_vm(kLoads));
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < kRd; ++i) rd(0, 0, 0, i);
  wait(0);
  __builtin_amdgcn_sched_barrier(0);

  uint32_t so = 0;  // the stage that holds the current slice
  for (;;) {
    int split, batch, m0, n0;
    place<kTM, kTN, kPairs>(g, p, split, batch, m0, n0);
    const int n_it = min(g.per, g.slices - split * g.per);
    f32x16 acc[kMB][kNB];
#pragma unroll
    for (int i = 0; i < kMB; ++i)
#pragma unroll
      for (int j = 0; j < kNB; ++j) acc[i][j] = f32x16{};
    for (int it = 0; it < n_it; ++it) {
      const uint32_t no = kStage - so;
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        const int z = kk & 1;
        bool late = false;  // loads already issued, before the products
        if (kk == 3) {
          __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));  // this wave's loads of the next slice are in LDS
          __builtin_amdgcn_s_barrier();               // every wave's, and this slice's reads are done
          __builtin_amdgcn_sched_barrier(0);
          late = ragged();
          if (late) load_ragged(so ? 1 : 0);
        }
#pragma unroll
        for (int f = 0; f < kMf; ++f) {  // one MFMA, its share of the next step's reads and of the loads
#pragma unroll
          for (int i = f * kRd / kMf; i < (f + 1) * kRd / kMf; ++i) {
            if (kk < 3) rd(z ^ 1, so, kk + 1, i);
            else rd(z ^ 1, no, 0, i);
          }
          if (kk == 3 && !late) {
#pragma unroll
            for (int j = f * kLoads / kMf; j < (f + 1) * kLoads / kMf; ++j) load(so ? 1 : 0, j);
          }
          const int jj = f / kNB, ii = f % kNB;
          acc[jj][ii] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(bfrag(z, ii), afrag(z, jj), acc[jj][ii], 0, 0, 0);
          __builtin_amdgcn_sched_barrier(0);
        }
        wait(z ^ 1);
        __builtin_amdgcn_sched_barrier(0);
      }
      advance();
      so = no;
    }
    if (g.partial) {
      f32x4* dst = reinterpret_cast<f32x4*>(g.partial) +
                   (static_cast<int64_t>(p) * 8 + wave) * (kMB * kNB * 4 * 64) + lane;
#pragma unroll
      for (int jj = 0; jj < kMB; ++jj)
#pragma unroll
        for (int ii = 0; ii < kNB; ++ii)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            dst[((jj * kNB + ii) * 4 + q) * 64] = f32x4{acc[jj][ii][4 * q], acc[jj][ii][4 * q + 1],
                                                        acc[jj][ii][4 * q + 2], acc[jj][ii][4 * q + 3]};
    } else {
      finish<kMode, C::kHalves>(acc, batch, m0 + wm * kMB * 32, n0 + wn * (kPairs ? 32 : 32 * kNB), lane,
                                lds0 + 2 * kStage + wave * C::kStrip);
    }
    p += g.wpx;
    if (p >= pend) break;
  }
  __builtin_amdgcn_s_waitcnt(0);  // the reload of the last slice
#undef TM_RD
#undef TM_TR
}

// The partial tiles of split s of tile t are at position s T + t, in the order of the accumulators
// (a wave's 64 lanes of one register group consecutive): summed split 0 first, then the strip's end.
template <int kMB, int kNB, int kMode>
__global__ __launch_bounds__(256) void lin_finish_kernel(const Args g) {
  using C = Tile<kMB, kNB>;
  __shared__ __attribute__((aligned(1024))) uint8_t strips[4 * C::kStrip];
  const int lane = threadIdx.x & 63;
  const int w4 = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int T = g.tiles_m * g.tiles_n * g.batch;
  const int id = static_cast<int>(blockIdx.x) * 4 + w4;  // (tile, wave, jj)
  const int t = id / (8 * kMB);
  if (t >= T) return;
  const int wave = (id / kMB) % 8, jj = id % kMB;
  int split, batch, m0, n0;
  place<C::kTM, C::kTN, kMode == kGate>(g, t, split, batch, m0, n0);
  constexpr int kVec = kNB * 4;
  const f32x4* src = reinterpret_cast<const f32x4*>(g.partial) +
                     (static_cast<int64_t>(t) * 8 + wave) * (kMB * kNB * 4 * 64) + jj * kVec * 64 + lane;
  const int64_t step = static_cast<int64_t>(T) * 8 * (kMB * kNB * 4 * 64);
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
  f32x16 v[1][kNB];
#pragma unroll
  for (int ii = 0; ii < kNB; ++ii)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      v[0][ii][4 * q] = sum[ii * 4 + q].x;
      v[0][ii][4 * q + 1] = sum[ii * 4 + q].y;
      v[0][ii][4 * q + 2] = sum[ii * 4 + q].z;
      v[0][ii][4 * q + 3] = sum[ii * 4 + q].w;
    }
  const int wm = wave >> 2, wn = wave & 3;
  finish<kMode, C::kHalves>(v, batch, m0 + (wm * kMB + jj) * 32, n0 + wn * (kMode == kGate ? 32 : 32 * kNB), lane,
                            static_cast<uint32_t>(reinterpret_cast<uintptr_t>(strips)) + w4 * C::kStrip);
}

// ------------------------------------------------------------------------------ the host's side

constexpr int64_t kMaxPartialBytes = int64_t(2) << 30;
// Measured on MI355X: microseconds of a 64-deep K slice of a 256 x 256 tile; of a 128 x 128 tile alone on
// its CU and of two of them on one; what a tile's end costs beyond its products.
constexpr double kUsSlice256 = 1.42, kUsSlice128 = 0.62, kUsSlice128Pair = 0.95;
constexpr double kUsLaunch = 3.0, kUsEnd = 2.0, kUsReduce = 3.0, kBytesPerUs = 4.5e6;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// What a call computes, in the kernel's terms.
struct Product {
  int64_t m, n, slices, batch;
  bool gate;  // n counts features, a tile has half as many as columns
};

struct Plan {
  int mb, nb;      // tile of 64 mb x 128 nb
  int64_t splits;
  double us;
};

Plan plan_of(const Product& q, int mb, int nb, int64_t splits) {
  const int64_t tm = 64 * mb, tn = 128 * nb / (q.gate ? 2 : 1);
  const int64_t tiles = ceil_div(q.m, tm) * ceil_div(q.n, tn) * q.batch, wgs = tiles * splits;
  const int64_t per = ceil_div(q.slices, splits);
  double us = kUsLaunch;
  if (mb == 4) us += ceil_div(wgs, 256) * (per * kUsSlice256 + kUsEnd);
  else if (nb == 2) us += ceil_div(wgs, 256) * (per * 0.5 * (kUsSlice256 + kUsSlice128) + kUsEnd);
  else if (wgs <= 256) us += per * kUsSlice128 + kUsEnd;
  else us += ceil_div(wgs, 512) * (per * kUsSlice128Pair + kUsEnd);
  if (splits > 1) us += kUsReduce + static_cast<double>(wgs) * (tm * 128 * nb) * 8.0 / kBytesPerUs;
  return {mb, nb, splits, us};
}

// The tile and the number of splits with the least estimated time.
Plan best_plan(const Product& q) {
  Plan best = {0, 0, 0, 0.0};
  const int shapes[2][2] = {{4, 2}, {2, q.gate ? 2 : 1}};
  for (const auto& sh : shapes) {
    const int64_t tiles = ceil_div(q.m, 64 * sh[0]) * ceil_div(q.n, 128 * sh[1] / (q.gate ? 2 : 1)) * q.batch;
    for (int64_t s = 1; s <= 64 && s <= q.slices; ++s) {
      if (ceil_div(q.slices, ceil_div(q.slices, s)) != s) continue;  // some split would be empty
      if (s > 1 && tiles * s * (64 * sh[0]) * (128 * sh[1]) * 4 > kMaxPartialBytes) break;
      const Plan p = plan_of(q, sh[0], sh[1], s);
      if (best.splits == 0 || p.us < best.us) best = p;
    }
  }
  return best;
}

size_t partial_bytes(const Product& q, const Plan& p) {
  if (p.splits <= 1) return 0;
  const int64_t tiles = ceil_div(q.m, 64 * p.mb) * ceil_div(q.n, 128 * p.nb / (q.gate ? 2 : 1)) * q.batch;
  return static_cast<size_t>(tiles * p.splits) * (64 * p.mb) * (128 * p.nb) * sizeof(float);
}

Product product_of(int op, int64_t rows, int64_t inp, int64_t out, bool two) {
  switch (op) {
    case TM_LIN_FORWARD: return {rows, out, ceil_div(inp, kSliceK), 1, false};
    case TM_LIN_GATE: return {rows, out, ceil_div(inp, kSliceK), 1, true};
    case TM_LIN_GRAD_X: return {rows, inp, ceil_div(out, kSliceK) * (two ? 2 : 1), 1, false};
    case TM_LIN_GATE_GRAD: return {rows, inp, ceil_div(out, kSliceK), 1, false};
    default: return {out, inp, ceil_div(rows, kSliceK), two ? 2 : 1, false};
  }
}

constexpr int kMaxDevices = 64, kKernels = 10;
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

template <int kMB, int kNB, bool kAK, bool kBK, int kMode>
int launch(int which, Args& g, hipStream_t s) {
  using C = Tile<kMB, kNB>;
  int cus = 0;
  const void* fn = reinterpret_cast<const void*>(lin_kernel<kMB, kNB, kAK, kBK, kMode>);
  hipError_t e = allow_lds(s, which, fn, C::kLds, &cus);
  if (e != hipSuccess) return lin_fail(TM_ELAUNCH, "tm_lin: LDS attribute: %s", hipGetErrorString(e));
  const int64_t positions = static_cast<int64_t>(g.tiles_m) * g.tiles_n * g.batch * g.splits;
  const int64_t per_xcd = ceil_div(positions, 8), room = (cus >= 16 ? cus / 8 : 1) * (2 * C::kLds <= 163840 ? 2 : 1);
  g.wpx = static_cast<int>(per_xcd < room ? per_xcd : room);
  hipLaunchKernelGGL((lin_kernel<kMB, kNB, kAK, kBK, kMode>), dim3(static_cast<uint32_t>(8 * g.wpx)), dim3(512), C::kLds,
                     s, g);
  e = hipGetLastError();
  if (e != hipSuccess) return lin_fail(TM_ELAUNCH, "lin_kernel: launch failed: %s", hipGetErrorString(e));
  if (g.splits > 1) {
    const int64_t waves = positions / g.splits * 8 * kMB;
    hipLaunchKernelGGL((lin_finish_kernel<kMB, kNB, kMode>), dim3(static_cast<uint32_t>(ceil_div(waves, 4))), dim3(256),
                       0, s, g);
    e = hipGetLastError();
    if (e != hipSuccess) return lin_fail(TM_ELAUNCH, "lin_finish_kernel: launch failed: %s", hipGetErrorString(e));
  }
  return TM_OK;
}

}  // namespace

extern "C" {

size_t tm_lin_workspace_bytes(int op, int64_t rows, int64_t inp, int64_t out, int two) {
  if (op < TM_LIN_FORWARD || op > TM_LIN_GRAD_W || rows <= 0 || inp <= 0 || out <= 0) return 0;
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
  const size_t need = partial_bytes(q, p);
  if (need && (!d_ws || ws_bytes < need || !aligned(d_ws, 16)))
    return lin_fail(TM_EINVAL, "tm_lin: workspace of %zu bytes, %zu needed, 16-byte aligned", ws_bytes, need);
  auto up8 = [](int64_t v) { return (v + 7) / 8 * 8; };
  // the stored widths of the operands, and what of K each holds
  const int64_t wide_a = op == TM_LIN_FORWARD || op == TM_LIN_GATE ? up8(d->inp)
                         : op == TM_LIN_GRAD_X && two              ? 2 * ceil_div(d->out, kSliceK) * kSliceK
                         : op == TM_LIN_GRAD_W && two_out          ? ceil_div(d->out, kSliceK) * kSliceK + up8(d->out)
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
      g.a_batch = ceil_div(d->out, kSliceK) * kSliceK * 2;
  }
  g.splits = static_cast<int>(p.splits);
  g.per = static_cast<int>(ceil_div(q.slices, p.splits));
  const int64_t tiles_m = ceil_div(q.m, 64 * p.mb), tiles_n = ceil_div(q.n, 128 * p.nb / (q.gate ? 2 : 1));
  if (tiles_m * tiles_n * q.batch * p.splits > (int64_t(1) << 27))
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
    const int64_t pad = op == TM_LIN_GATE ? up8(cols) : ceil_div(cols, kSliceK) * kSliceK;
    g.n_store = static_cast<int>(pad);
    if (g.out_f32 || d->ldo % 8 || d->ldo < (op == TM_LIN_GATE ? pad : 2 * pad) || !aligned(d->o0, 16) ||
        (op == TM_LIN_GATE_GRAD && d->o1 && (d->ldo1 % 8 || d->ldo1 < pad || !aligned(d->o1, 16))))
      return lin_fail(TM_EINVAL, "tm_lin: the gate's outputs are bf16, 16-byte aligned, rows %lld and %lld elements apart "
                      "a multiple of 8 that holds %lld columns each", (long long)d->ldo, (long long)d->ldo1,
                      (long long)pad);
  } else if (d->ldo < cols || (g.out_f32 && (!aligned(d->o0, 4) || !aligned(d->o1, 4)))) {
    return lin_fail(TM_EINVAL, "tm_lin: output rows %lld elements apart for %lld columns", (long long)d->ldo,
                    (long long)cols);
  }
  g.out_vec = d->ldo % (g.out_f32 ? 4 : 8) == 0 && aligned(d->o0, 16) && aligned(d->o1, 16);
  g.bias = static_cast<const char*>(d->bias);
  g.bias_f32 = d->bias_f32 != 0;
  g.bias_vec = aligned(d->bias, g.bias_f32 ? 16 : 8);
  g.res = static_cast<const char*>(d->res);
  g.res_f32 = d->res_f32 != 0;
  g.ldr = d->ldr;
  g.res_vec = d->ldr % (g.res_f32 ? 4 : 8) == 0 && aligned(d->res, 16);

  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool big = p.mb == 4;
  switch (op) {
    case TM_LIN_FORWARD:
      return big ? launch<4, 2, true, true, kLinear>(0, g, s) : launch<2, 1, true, true, kLinear>(1, g, s);
    case TM_LIN_GATE:
      return big ? launch<4, 2, true, true, kGate>(2, g, s) : launch<2, 2, true, true, kGate>(3, g, s);
    case TM_LIN_GRAD_X:
      return big ? launch<4, 2, true, false, kPlain>(4, g, s) : launch<2, 1, true, false, kPlain>(5, g, s);
    case TM_LIN_GATE_GRAD:
      return big ? launch<4, 2, true, false, kGateGrad>(6, g, s) : launch<2, 1, true, false, kGateGrad>(7, g, s);
    default:
      return big ? launch<4, 2, false, false, kPlain>(8, g, s) : launch<2, 1, false, false, kPlain>(9, g, s);
  }
}

}  // extern "C"
