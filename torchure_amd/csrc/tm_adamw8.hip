// tm_adamw8.hip -- gfx950 kernels of the AdamW step on moments held in 8 bits.
//
// What is held. A tensor's elements, in order, are cut into blocks of 64. The first moment m is held as e4m3 values with a
// power of two for each block (the byte e + 127; e as in tm_act.h). Of the second moment the root r is held, which is what
// the step divides by, as n(c) 2^x: c is 8 bits without a sign, n(c) = c below 16, else
// (16 + c % 16) 2^(c / 16 - 1), 254 the largest code of a number and 255 NaN; x is the least with which the block's largest finite r is at
// most n(254) 2^x, at least -105 (the byte x + 145). A step of r is 1/16 to 1/32 of it down to 2^-15 of the block's largest, and
// a nonzero r is never held as 0, which would leave a step divided by eps alone.
//
// Rounding is stochastic: a moment moves by (1 - beta) of its distance to the new gradient in a step, less than half a
// step of 8 bits (2^-4 of m, 2^-5 of r) for most, and to the nearest it would stay where it is for ever (beta2 = 0.999: r moves by
// 5e-4 of itself). Rounded up with the probability of the part that lies above, what is held has the right mean.
// The random bits are a hash of (seed, step, element): the same run gives the same bits, on any launch shape. The tensor has no part in
// it: elements i of all tensors are rounded by the same bits in a step.
//
// The new moments are summed in fp64 as in the 32-bit step and rounded to fp32 once (sums in fp32 turned three times as many of the
// roundings the other way); the rest is fp32. Which way a root is rounded goes by its sum in fp64 too. The step uses the moments before
// they are held again.
//
// Bound by memory: 16.06 bytes a param with bf16 grads and copies (28 with 32-bit moments). The codes were computed with per-value
// tests, selects and e4m3 conversions first, 300 vector instructions a wave, which bound the step at 5.5 TB/s; as float's own denormals
// (below) it runs at 5.7-5.95, in-order streams of 256 to 1024 bytes a wave.

#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>
#include <string.h>

#include <algorithm>

#include "torchure_amd.h"
#include "tm_act.h"
#include "tm_internal.h"

namespace {

using tm_act::bf16_hi;
using tm_act::bf16_lo;
using tm_act::f32x4;
using tm_act::pack_bf16;
using tm_act::u32x2;

typedef uint32_t u32_at1 __attribute__((aligned(1)));
typedef u32x2 u32x2_at2 __attribute__((aligned(2)));
typedef f32x4 f32x4_at4 __attribute__((aligned(4)));

template <typename... A>
int fail(int code, const char* fmt, A... args) {
  return tm_internal_fail(code, fmt, args...);
}

constexpr int kThreads = 256;
constexpr int kWave = 64;
constexpr int kSlice = kWave * 4;  // elements a wave takes at a time: four blocks, 16 lanes each
constexpr int kBlock = 64;
// Slices to a wave: the step's eight streams are fastest with one (5.95 TB/s over 2e9 elements, 5.75 with two, 5.95
// with four and twice the registers; a cap on the waves of a CU, as the 32-bit step has, only loses), reading
// the moments' two streams in and two out with two (6.16 TB/s, one 5.6, four 5.6).
constexpr int kStepSlices = 1, kReadSlices = 2;
static_assert(TM_CHUNK_ALIGN % (kSlice * kStepSlices) == 0 && TM_CHUNK_ALIGN % (kSlice * kReadSlices) == 0, "whole pieces to a chunk");
constexpr int kRootLow = 40;  // the least byte of a root's exponent

// Global-address-space accesses, past the caches: every byte is touched once. (Cached loads or stores in the step: 5.5 TB/s;
// the codes that moments8_kernel reads alone are faster through them, 6.16 TB/s for 5.85.)
#define TM_GLOBAL __attribute__((address_space(1)))
// (Types of their elements' alignment; a template's argument would lose it.)
template <bool kCached>
__device__ __forceinline__ uint32_t load_bytes(const uint8_t* p) {
  const auto* q = (const TM_GLOBAL u32_at1*)p;
  return kCached ? *q : __builtin_nontemporal_load(q);
}
__device__ __forceinline__ void store_bytes(uint8_t* p, uint32_t v) {
  __builtin_nontemporal_store(static_cast<u32_at1>(v), (TM_GLOBAL u32_at1*)p);
}

// ---------------------------------------------------------------- random bits

// A: the prime nearest to 2^32 over the golden ratio. B and C: of 400 random odd pairs the one with which, where a bit of the input turns,
// each bit of the output turns nearest to half the time.
constexpr uint32_t kHashA = 0x9E3779B1u, kHashB = 0x8C2549D1u, kHashC = 0xD406A25Du;

__device__ __forceinline__ uint32_t mix(uint32_t z) {
  z = (z ^ (z >> 16)) * kHashB;
  z = (z ^ (z >> 15)) * kHashC;
  return z ^ (z >> 16);
}

// One multiplication an element: a bijection of i * A + key, so each half is uniform over any 2^32 of them. (Measured over
// 2^20 neighbours and over 2^16 steps of one element: means within 5e-4, correlations of neighbours,
// steps and halves below 0.008.)
__device__ __forceinline__ uint32_t element_bits(uint32_t z) {
  z = (z ^ (z >> 16)) * kHashB;
  return z ^ (z >> 15);
}

// ---------------------------------------------------------------- the two formats
//
// Both are the top bits of a float that is scaled so that the format's smallest normal number is float's own, 2^-126:
// below, float's denormals have the format's constant step. A code is then (bits + random bits below the last place) >> the
// places left out, and a value the float of the shifted code, scaled back. (ldexp: the scales pass 2^127.)

__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7FFFFFFFu) < 0x7F800000u; }

// e4m3: 2^-6 2^e -> 2^-126. Root: 16 2^x -> 2^-126, x = byte - 145.
__device__ __forceinline__ float scale_m(float m, uint32_t me) { return ldexpf(m, 7 - static_cast<int>(me)); }
__device__ __forceinline__ float scale_root(float r, uint32_t re) { return ldexpf(r, 15 - static_cast<int>(re)); }

// Up where the part above the lower code plus u is at least 1, u = (16 random bits + 1/2) / 2^16; m's are the low
// ones of `bits`, a root's the high ones. kAny: values that are infinite, NaN or past what can be held.
template <bool kAny>
__device__ __forceinline__ uint32_t hold_m(float m, uint32_t me, uint32_t bits) {
  float y = scale_m(m, me);
  if constexpr (kAny) y = __builtin_amdgcn_fmed3f(y, -0x1.cp-112f, 0x1.cp-112f);  // 448 2^-120
  const uint32_t up = __float_as_uint(y) + ((bits & 0xFFFFu) << 4 | 8u);
  const uint32_t c = (up >> 24 & 0x80u) | (up >> 20 & 0x7Fu);
  return kAny && !finite(m) ? 0x7Fu : c;
}
// A root has no sign, which would reach the next element's code. `up`: its code and the bits below, the random ones added.
__device__ __forceinline__ uint32_t root_up(float r, uint32_t re, uint32_t bits) {
  return __float_as_uint(scale_root(r, re)) + ((bits >> 13 & ~7u) | 4u);
}
template <bool kAny>
__device__ __forceinline__ uint32_t hold_root(float r, uint32_t up) {
  const uint32_t c = max(up >> 19, min(__float_as_uint(r), 1u));
  return kAny && !finite(r) ? 255u : c;
}
__device__ __forceinline__ float read_root(uint32_t c, uint32_t re) {
  return ldexpf(__uint_as_float(c << 19), static_cast<int>(re) - 15);
}

// Four elements of a lane, its block's exponents in all 16 lanes of a row.
struct Codes {
  uint32_t m, r;     // a byte an element
  uint32_t me, re;   // the exponents' bytes
};

// past(j): whether r[j] is past the root that it was rounded from. The places at which a root turns are fp32 numbers, and half of those
// just below one are rounded onto it (510 to 560 of 574e6 were held otherwise than in 64 bits, none so). Looked at where a root lies on one,
// which one wave in 2000 sees: for each root it cost the step 1-1.6%, so nothing; exp_avg's values (14-25 of 37e6 with fp32 gradients, none
// with bf16 ones) in the same way 1-2%, for want of registers.
template <bool kAny, class Past>
__device__ __forceinline__ void codes4(Codes& c, const float* m, const float* r, const uint32_t* bits, Past&& past) {
  uint32_t up[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) up[j] = root_up(r[j], c.re, bits[j]);
  if (min(min(up[0] << 13, up[1] << 13), min(up[2] << 13, up[3] << 13)) == 0) {
#pragma unroll
    for (int j = 0; j < 4; ++j) up[j] -= past(j);
  }
  c.m = c.r = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    c.m |= hold_m<kAny>(m[j], c.me, bits[j]) << (8 * j);
    c.r |= hold_root<kAny>(r[j], up[j]) << (8 * j);
  }
}

__device__ __forceinline__ uint32_t most4(const float* x) {
  return max(max(__float_as_uint(x[0]) & 0x7FFFFFFFu, __float_as_uint(x[1]) & 0x7FFFFFFFu),
             max(__float_as_uint(x[2]) & 0x7FFFFFFFu, __float_as_uint(x[3]) & 0x7FFFFFFFu));
}

template <class Past>
__device__ __forceinline__ Codes hold4(const float* m, const float* r, const uint32_t* bits, Past&& past) {
  Codes c;
  uint32_t most_m = most4(m), most_r = most4(r);
  // a wave with an m past all blocks' range, an infinity or a NaN looks at each value
  const bool any = __any(max(most_m, most_r) > tm_act::kPlainMost);
  if (any) {
    most_m = tm_act::largest_finite<4>(m);
    most_r = tm_act::largest_finite<4>(r);
  }
  most_m = tm_act::row_max(most_m);
  most_r = tm_act::row_max(most_r);
  c.me = static_cast<uint32_t>(tm_act::block_exponent(most_m) + 127);
  c.re = max((most_r + 0x000FFFFFu) >> 23, static_cast<uint32_t>(kRootLow));
  if (any) codes4<true>(c, m, r, bits, past);
  else codes4<false>(c, m, r, bits, past);
  return c;
}

__device__ __forceinline__ void read4(const Codes& c, float* m, float* r) {
  const f32x4 d = tm_act::decode4(c.m, tm_act::two_to(static_cast<int>(c.me) - 127));
  m[0] = d.x; m[1] = d.y; m[2] = d.z; m[3] = d.w;
#pragma unroll
  for (int j = 0; j < 4; ++j) r[j] = read_root((c.r >> (8 * j)) & 0xFFu, c.re);
  if (__any(((~c.r - 0x01010101u) & c.r & 0x80808080u) != 0)) {  // a byte of 255
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (((c.r >> (8 * j)) & 0xFFu) == 255u) r[j] = __uint_as_float(0x7FC00000u);
  }
}

// A tensor's held moment: codes of all elements up to the next multiple of 256, then the blocks' exponents.
__device__ __host__ __forceinline__ int64_t held_codes(int64_t n) { return (n + kSlice - 1) / kSlice * kSlice; }

template <bool kCached = false>
__device__ __forceinline__ Codes load_codes(const tm_tensor_t& d, int64_t codes, int64_t e) {
  const uint8_t* m = reinterpret_cast<const uint8_t*>(d.exp_avg);
  const uint8_t* r = reinterpret_cast<const uint8_t*>(d.exp_avg_sq);
  return {load_bytes<kCached>(m + e), load_bytes<kCached>(r + e), m[codes + e / kBlock], r[codes + e / kBlock]};
}
__device__ __forceinline__ void store_codes(const tm_tensor_t& d, int64_t codes, int64_t e, const Codes& c) {
  uint8_t* m = reinterpret_cast<uint8_t*>(d.exp_avg);
  uint8_t* r = reinterpret_cast<uint8_t*>(d.exp_avg_sq);
  store_bytes(m + e, c.m);
  store_bytes(r + e, c.r);
  if ((threadIdx.x & 15) == 0) {
    m[codes + e / kBlock] = static_cast<uint8_t>(c.me);
    r[codes + e / kBlock] = static_cast<uint8_t>(c.re);
  }
}

// Four values from element e on, `left` of them there (0 to 4; zeros after): whole vectors at any element's alignment.
// kWhole: all are.
template <bool kWhole>
__device__ __forceinline__ void load_f32(float* v, uint64_t base, int64_t e, int left) {
  const float* p = reinterpret_cast<const float*>(base) + e;
  if (kWhole || left == 4) {
    const f32x4 a = __builtin_nontemporal_load((const TM_GLOBAL f32x4_at4*)p);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = j < left ? p[j] : 0.0f;
  }
}
template <bool kWhole>
__device__ __forceinline__ void store_f32(uint64_t base, int64_t e, int left, const float* v) {
  float* p = reinterpret_cast<float*>(base) + e;
  if (kWhole || left == 4) {
    const f32x4_at4 a = f32x4{v[0], v[1], v[2], v[3]};
    __builtin_nontemporal_store(a, (TM_GLOBAL f32x4_at4*)p);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < left) p[j] = v[j];
  }
}
template <bool kWhole>
__device__ __forceinline__ void load_bf16(float* v, uint64_t base, int64_t e, int left) {
  const uint16_t* p = reinterpret_cast<const uint16_t*>(base) + e;
  if (kWhole || left == 4) {
    const u32x2 w = __builtin_nontemporal_load((const TM_GLOBAL u32x2_at2*)p);
    v[0] = bf16_lo(w.x); v[1] = bf16_hi(w.x); v[2] = bf16_lo(w.y); v[3] = bf16_hi(w.y);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = j < left ? bf16_lo(p[j]) : 0.0f;
  }
}
template <bool kWhole>
__device__ __forceinline__ void store_bf16(uint64_t base, int64_t e, int left, const float* v) {
  uint16_t* p = reinterpret_cast<uint16_t*>(base) + e;
  const u32x2_at2 w = u32x2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
  if (kWhole || left == 4) {
    __builtin_nontemporal_store(w, (TM_GLOBAL u32x2_at2*)p);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < left) p[j] = static_cast<uint16_t>((j < 2 ? w.x : w.y) >> (16 * (j & 1)));
  }
}

// This workgroup's chunk, and the first element of its kSlices slices, in the table's order. (A power of two takes a shift for the
// division's 25 instructions. Neighbouring slices run on different XCDs, each of which reads and writes part of
// an exponents' line: 1.028 times the bytes. 32 slices in a row to an XCD had whole lines and were 9% slower.)
template <int kSlices>
__device__ __forceinline__ int64_t piece_of(const tm_chunk_t* __restrict__ chunks, uint32_t first_chunk,
                                            uint32_t pieces_per_chunk, int64_t chunk_elems, tm_chunk_t& ck) {
  const bool pow2 = (pieces_per_chunk & (pieces_per_chunk - 1)) == 0;
  const uint32_t local = pow2 ? blockIdx.x >> __builtin_ctz(pieces_per_chunk) : blockIdx.x / pieces_per_chunk;
  ck = chunks[first_chunk + local];
  return static_cast<int64_t>(ck.chunk) * chunk_elems +
         static_cast<int64_t>(blockIdx.x - local * pieces_per_chunk) * (kSlices * kSlice);
}

// How many of the four elements from e on there are.
__device__ __forceinline__ int left_of(int64_t numel, int64_t e) {
  return static_cast<int>(max(int64_t(0), min(int64_t(4), numel - e)));
}

// ---------------------------------------------------------------- the step

// What the update needs of a tensor, made once for it (64 bytes, in the workspace).
struct alignas(16) Scal {
  double beta1, omb1, beta2, omb2;
  float neg_lrwd, eps, step_size, inv_bc2s;
  uint32_t key, flags, pad[2];
};
constexpr uint32_t kDecay = 1u, kF32 = 2u, kOut = 4u, kClip = 8u;

struct Hyper {
  tm_hyper_t g[TM_MAX_GROUPS];
  int32_t n;
};

__global__ __launch_bounds__(kThreads) void adamw8_prep_kernel(const tm_tensor_t* __restrict__ tensors, int64_t n_tensors,
                                                               Hyper hyper, uint32_t seed_lo, uint32_t seed_hi,
                                                               Scal* __restrict__ scal) {
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (t >= n_tensors) return;
  const tm_tensor_t d = tensors[t];
  float* step_p = reinterpret_cast<float*>(d.step);
  Scal s = {};
  s.flags = ((d.flags & TM_GRAD_F32) ? kF32 : 0u) | (d.param_bf16 ? kOut : 0u) | ((d.flags & TM_FLAG_CLIP) ? kClip : 0u);
  if (d.group < 0 || d.group >= hyper.n) {
    // as in the 32-bit step: a record naming a group that the call does not have is poisoned
    const float nan = __builtin_nanf("");
    *step_p = nan;
    s.beta1 = s.omb1 = s.beta2 = s.omb2 = nan;
    s.neg_lrwd = s.eps = s.step_size = s.inv_bc2s = nan;
    s.flags |= kDecay;
    scal[t] = s;
    return;
  }
  const tm_hyper_t h = hyper.g[d.group];
  const float step = *step_p + 1.0f;
  *step_p = step;
  const double bc1 = 1.0 - pow(h.beta1, static_cast<double>(step));
  const double bc2 = 1.0 - pow(h.beta2, static_cast<double>(step));
  s.neg_lrwd = static_cast<float>(-(h.lr * h.weight_decay));
  s.beta1 = h.beta1;
  s.omb1 = 1.0 - h.beta1;
  s.beta2 = h.beta2;
  s.omb2 = 1.0 - h.beta2;
  s.eps = static_cast<float>(h.eps);
  s.step_size = static_cast<float>(h.lr / bc1);
  s.inv_bc2s = static_cast<float>(1.0 / sqrt(bc2));
  s.flags |= h.weight_decay != 0.0 ? kDecay : 0u;
  s.key = mix(static_cast<uint32_t>(fminf(step, 4.0e9f)) + mix(seed_hi + mix(seed_lo)));
  scal[t] = s;
}

// A wave's kStepSlices slices from `start` on: 4 elements a lane of each, a block of 64 to 16 lanes, whose largest moments meet
// by DPP moves.
template <bool kF32, bool kWhole>
__device__ __forceinline__ void update(const tm_tensor_t& d, const Scal& s, float coef, int64_t start) {
  const int64_t e0 = start + static_cast<int64_t>(threadIdx.x) * 4, codes = held_codes(d.numel);
  float p[kStepSlices][4], g[kStepSlices][4];
  Codes was[kStepSlices];
#pragma unroll
  for (int k = 0; k < kStepSlices; ++k) {
    const int64_t e = e0 + k * kSlice;
    if (!kWhole && start + k * kSlice >= d.numel) continue;  // else the slice's codes are there, all of them
    const int left = kWhole ? 4 : left_of(d.numel, e);
    if constexpr (kF32) load_f32<kWhole>(g[k], d.grad, e, left);
    else load_bf16<kWhole>(g[k], d.grad, e, left);
    load_f32<kWhole>(p[k], d.master, e, left);
    was[k] = load_codes(d, codes, e);
  }
#pragma unroll
  for (int k = 0; k < kStepSlices; ++k) {
    const int64_t e = e0 + k * kSlice;
    if (!kWhole && start + k * kSlice >= d.numel) continue;
    float m[4], r[4];
    read4(was[k], m, r);
    uint32_t bits[4];
    double v[4];
    const uint32_t z = static_cast<uint32_t>(e) * kHashA + s.key;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float gj = g[k][j] * coef;
      const float pj = (s.flags & kDecay) ? fmaf(s.neg_lrwd, p[k][j], p[k][j]) : p[k][j];
      const double gd = gj;
      m[j] = static_cast<float>(fma(s.beta1, static_cast<double>(m[j]), s.omb1 * gd));
      v[j] = fma(s.beta2, static_cast<double>(r[j] * r[j]), s.omb2 * gd * gd);
      r[j] = sqrtf(static_cast<float>(v[j]));
      p[k][j] = pj - s.step_size * m[j] / fmaf(r[j], s.inv_bc2s, s.eps);
      bits[j] = element_bits(z + j * kHashA);
    }
    const Codes now = hold4(m, r, bits, [&](int j) { return fma(-static_cast<double>(r[j]), static_cast<double>(r[j]), v[j]) < 0.0; });
    const int left = kWhole ? 4 : left_of(d.numel, e);
    store_f32<kWhole>(d.master, e, left, p[k]);
    store_codes(d, codes, e, now);
    if (s.flags & kOut) store_bf16<kWhole>(d.param_bf16, e, left, p[k]);
  }
}

__global__ __launch_bounds__(kWave) void adamw8_update_kernel(const tm_tensor_t* __restrict__ tensors, int64_t n_tensors,
                                                              const tm_chunk_t* __restrict__ chunks, uint32_t first_chunk,
                                                              uint32_t pieces_per_chunk, int64_t chunk_elems,
                                                              const Scal* __restrict__ scal,
                                                              const float* __restrict__ coef_p) {
  tm_chunk_t ck;
  const int64_t start = piece_of<kStepSlices>(chunks, first_chunk, pieces_per_chunk, chunk_elems, ck);
  if (ck.tensor >= n_tensors) return;
  const tm_tensor_t d = tensors[ck.tensor];
  if (start >= d.numel) return;
  const Scal s = scal[ck.tensor];
  const float coef = (s.flags & kClip) && coef_p ? *coef_p : 1.0f;
  const bool whole = start + kStepSlices * kSlice <= d.numel;
  if (s.flags & kF32) {
    if (whole) update<true, true>(d, s, coef, start);
    else update<true, false>(d, s, coef, start);
  } else {
    if (whole) update<false, true>(d, s, coef, start);
    else update<false, false>(d, s, coef, start);
  }
}

// ---------------------------------------------------------------- moments as values

// kRead: master = exp_avg's values and grad = the root's, in bf16, or with TM_GRAD_F32 exp_avg's and exp_avg_sq's
// (the root's square) in fp32. Else the fp32 exp_avg and exp_avg_sq there are held, to the nearest.
template <bool kRead, bool kWhole>
__device__ __forceinline__ void move_moments(const tm_tensor_t& d, int64_t start) {
  const int64_t e0 = start + static_cast<int64_t>(threadIdx.x) * 4, codes = held_codes(d.numel);
  Codes was[kReadSlices];
  if constexpr (kRead) {
#pragma unroll
    for (int k = 0; k < kReadSlices; ++k)
      if (kWhole || start + k * kSlice < d.numel) was[k] = load_codes<true>(d, codes, e0 + k * kSlice);
  }
#pragma unroll
  for (int k = 0; k < kReadSlices; ++k) {
    const int64_t e = e0 + k * kSlice;
    if (!kWhole && start + k * kSlice >= d.numel) continue;
    const int left = kWhole ? 4 : left_of(d.numel, e);
    float m[4], r[4];
    if constexpr (kRead) {
      read4(was[k], m, r);
      if (d.flags & TM_GRAD_F32) {
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] *= r[j];
        store_f32<kWhole>(d.master, e, left, m);
        store_f32<kWhole>(d.grad, e, left, r);
      } else {
        store_bf16<kWhole>(d.master, e, left, m);
        store_bf16<kWhole>(d.grad, e, left, r);
      }
    } else {
      load_f32<kWhole>(m, d.master, e, left);
      load_f32<kWhole>(r, d.grad, e, left);
#pragma unroll
      for (int j = 0; j < 4; ++j) r[j] = fabsf(sqrtf(r[j]));  // (the root of -0 is -0)
      const uint32_t half[4] = {0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u};
      store_codes(d, codes, e, hold4(m, r, half, [](int) { return false; }));
    }
  }
}

template <bool kRead>
__global__ __launch_bounds__(kWave) void moments8_kernel(const tm_tensor_t* __restrict__ tensors, int64_t n_tensors,
                                                         const tm_chunk_t* __restrict__ chunks, uint32_t first_chunk,
                                                         uint32_t pieces_per_chunk, int64_t chunk_elems) {
  tm_chunk_t ck;
  const int64_t start = piece_of<kReadSlices>(chunks, first_chunk, pieces_per_chunk, chunk_elems, ck);
  if (ck.tensor >= n_tensors) return;
  const tm_tensor_t d = tensors[ck.tensor];
  if (start >= d.numel) return;
  if (start + kReadSlices * kSlice <= d.numel) move_moments<kRead, true>(d, start);
  else move_moments<kRead, false>(d, start);
}

// kernel(first_chunk, pieces_per_chunk, blocks) over a chunk table, a piece of `slices` slices to a workgroup: launches of
// less than 2^32 work-items, of whole chunks.
template <class F>
int launch_chunks(int64_t n_chunks, int64_t chunk_elems, int slices, const char* what, F&& launch) {
  const int64_t spc = chunk_elems / (kSlice * slices), per = 0xFFFFFFFFll / kWave / spc;
  for (int64_t first = 0; first < n_chunks; first += per) {
    const int64_t cnt = std::min(per, n_chunks - first);
    launch(static_cast<uint32_t>(first), static_cast<uint32_t>(spc), dim3(static_cast<uint32_t>(cnt * spc)));
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return fail(TM_ELAUNCH, "%s: launch failed: %s", what, hipGetErrorString(err));
  }
  return TM_OK;
}

template <bool kRead>
int moments8(const tm_tensor_t* d_tensors, int64_t n_tensors, const tm_chunk_t* d_chunks, int64_t n_chunks,
             int64_t chunk_elems, void* stream, const char* who) {
  const int rc = tm_internal_check_table(d_tensors, n_tensors, d_chunks, n_chunks, chunk_elems, who);
  if (rc) return rc;
  return launch_chunks(n_chunks, chunk_elems, kReadSlices, who, [&](uint32_t first, uint32_t spc, dim3 grid) {
    hipLaunchKernelGGL(moments8_kernel<kRead>, grid, dim3(kWave), 0, static_cast<hipStream_t>(stream), d_tensors, n_tensors,
                       d_chunks, first, spc, chunk_elems);
  });
}

}  // namespace

extern "C" {

int64_t tm_moments8_bytes(int64_t numel) { return numel <= 0 ? 0 : held_codes(numel) + held_codes(numel) / kBlock; }

int tm_adamw8_step(const tm_tensor_t* d_tensors, int64_t n_tensors, const tm_chunk_t* d_chunks, int64_t n_chunks,
                   int64_t chunk_elems, const tm_hyper_t* h_groups, int32_t n_groups, const float* d_coef, uint64_t seed,
                   void* d_ws, void* stream) {
  const char* who = "tm_adamw8_step";
  int rc = tm_internal_check_table(d_tensors, n_tensors, d_chunks, n_chunks, chunk_elems, who);
  if (rc) return rc;
  if (n_groups < 1 || n_groups > TM_MAX_GROUPS || !h_groups)
    return fail(TM_EINVAL, "%s: n_groups %d outside 1..%d", who, n_groups, TM_MAX_GROUPS);
  if (!d_ws) return fail(TM_EINVAL, "%s: null workspace", who);
  if (n_tensors == 0) return TM_OK;
  Hyper hyper;
  memset(&hyper, 0, sizeof(hyper));
  for (int i = 0; i < n_groups; ++i) hyper.g[i] = h_groups[i];
  hyper.n = n_groups;
  // where the 32-bit step keeps its constants too: behind the norm's partial sums
  Scal* scal = reinterpret_cast<Scal*>(static_cast<char*>(d_ws) + sizeof(double) * TM_NORM_PARTIALS);
  static_assert(sizeof(Scal) == 64, "tm_workspace_bytes holds 64 bytes a tensor");
  hipStream_t s = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(adamw8_prep_kernel, dim3(static_cast<uint32_t>((n_tensors + kThreads - 1) / kThreads)), dim3(kThreads), 0,
                     s, d_tensors, n_tensors, hyper, static_cast<uint32_t>(seed), static_cast<uint32_t>(seed >> 32), scal);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return fail(TM_ELAUNCH, "adamw8_prep_kernel: launch failed: %s", hipGetErrorString(err));
  return launch_chunks(n_chunks, chunk_elems, kStepSlices, "adamw8_update_kernel", [&](uint32_t first, uint32_t spc, dim3 grid) {
    hipLaunchKernelGGL(adamw8_update_kernel, grid, dim3(kWave), 0, s, d_tensors, n_tensors, d_chunks, first, spc, chunk_elems,
                       scal, d_coef);
  });
}

int tm_moments8_read(const tm_tensor_t* d_tensors, int64_t n_tensors, const tm_chunk_t* d_chunks, int64_t n_chunks,
                     int64_t chunk_elems, void* stream) {
  return moments8<true>(d_tensors, n_tensors, d_chunks, n_chunks, chunk_elems, stream, "tm_moments8_read");
}

int tm_moments8_write(const tm_tensor_t* d_tensors, int64_t n_tensors, const tm_chunk_t* d_chunks, int64_t n_chunks,
                      int64_t chunk_elems, void* stream) {
  return moments8<false>(d_tensors, n_tensors, d_chunks, n_chunks, chunk_elems, stream, "tm_moments8_write");
}

}  // extern "C"
