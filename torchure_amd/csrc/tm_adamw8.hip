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
// The random bits are a hash of (seed, step, element): the same run gives the same bits, on any launch shape.
//
// Arithmetic is fp32 (the 32-bit step's is fp64, to the bit of torch's): errors of 1e-7 beside a held moment's 2^-4. The step uses the
// moments before they are rounded.

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
constexpr int kRootLow = 40;  // the least byte of a root's exponent

// Global-address-space accesses, past the caches: every byte is touched once.
#define TM_GLOBAL __attribute__((address_space(1)))
template <typename T>
__device__ __forceinline__ T ld(const void* p) {
  return __builtin_nontemporal_load((const TM_GLOBAL T*)p);
}
template <typename T, typename V>
__device__ __forceinline__ void st(void* p, V v) {
  __builtin_nontemporal_store(static_cast<T>(v), (TM_GLOBAL T*)p);
}

// ---------------------------------------------------------------- random bits

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

__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7FFFFFFFu) < 0x7F800000u; }

// m / 2^e to a whole number of e4m3 steps, up where the part above the lower one plus u is at least 1, u = (low 16
// of `bits` + 1/2) / 2^16. Below 2^-6 the step is 2^-9: adding 2^-6 puts the value into the binade of that step.
__device__ __forceinline__ float hold_m(float m, float inv, uint32_t bits) {
  const float y = m * inv, size = fminf(fabsf(y), 448.0f), base = size < 0x1p-6f ? 0x1p-6f : 0.0f;
  const uint32_t up = __float_as_uint(size + base) + ((bits & 0xFFFFu) * 16u + 8u);
  const float held = __uint_as_float(up & 0xFFF00000u) - base;
  return finite(m) ? copysignf(held, y) : __uint_as_float(0x7FC00000u);
}

// `k`: the exponent's byte. Numbers from 16 2^x on are floats whose top bits are the code; below, adding 16 2^x makes
// them so.
__device__ __forceinline__ uint32_t root_base(uint32_t k) { return (k - 15u) << 23; }
__device__ __forceinline__ uint32_t hold_root(float r, uint32_t k, uint32_t bits) {
  const uint32_t high = root_base(k), low = high + (1u << 23);
  const bool small = r < __uint_as_float(low);
  const uint32_t up = __float_as_uint(small ? r + __uint_as_float(low) : r) + ((bits >> 16) * 8u + 4u);
  const uint32_t c = (up >> 19) - ((small ? low : high) >> 19);
  return !finite(r) ? 255u : max(c, r > 0.0f ? 1u : 0u);
}
__device__ __forceinline__ float read_root(uint32_t c, uint32_t k) {
  const uint32_t high = root_base(k) + (c << 19), low = root_base(k) + (1u << 23);
  const float f = c < 16u ? __uint_as_float(high + (1u << 23)) - __uint_as_float(low) : __uint_as_float(high);
  return c == 255u ? __uint_as_float(0x7FC00000u) : f;
}

// Four elements of a lane, its block's exponents in all 16 lanes of a row.
struct Codes {
  uint32_t m, r;     // a byte an element
  uint32_t me, re;   // the exponents' bytes
};

__device__ __forceinline__ Codes hold4(const float* m, const float* r, const uint32_t* bits) {
  Codes c;
  const uint32_t most_m = tm_act::row_max(tm_act::largest_finite<4>(m));
  const uint32_t most_r = tm_act::row_max(tm_act::largest_finite<4>(r));
  const int e = tm_act::block_exponent(most_m);
  const float inv = tm_act::two_to(-e);
  c.me = static_cast<uint32_t>(e + 127);
  c.re = max((most_r + 0x000FFFFFu) >> 23, static_cast<uint32_t>(kRootLow));
  float h[4];
  c.r = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    h[j] = hold_m(m[j], inv, bits[j]);
    c.r |= hold_root(r[j], c.re, bits[j]) << (8 * j);
  }
  c.m = __builtin_amdgcn_cvt_pk_fp8_f32(h[0], h[1], 0, false);
  c.m = __builtin_amdgcn_cvt_pk_fp8_f32(h[2], h[3], c.m, true);
  return c;
}

__device__ __forceinline__ void read4(const Codes& c, float* m, float* r) {
  const f32x4 d = tm_act::decode4(c.m, tm_act::two_to(static_cast<int>(c.me) - 127));
  m[0] = d.x; m[1] = d.y; m[2] = d.z; m[3] = d.w;
#pragma unroll
  for (int j = 0; j < 4; ++j) r[j] = read_root((c.r >> (8 * j)) & 0xFFu, c.re);
}

// A tensor's held moment: codes of all elements up to the next multiple of 256, then the blocks' exponents.
__device__ __host__ __forceinline__ int64_t held_codes(int64_t n) { return (n + kSlice - 1) / kSlice * kSlice; }

__device__ __forceinline__ Codes load_codes(const tm_tensor_t& d, int64_t codes, int64_t e) {
  const uint8_t* m = reinterpret_cast<const uint8_t*>(d.exp_avg);
  const uint8_t* r = reinterpret_cast<const uint8_t*>(d.exp_avg_sq);
  return {ld<u32_at1>(m + e), ld<u32_at1>(r + e), m[codes + e / kBlock], r[codes + e / kBlock]};
}
__device__ __forceinline__ void store_codes(const tm_tensor_t& d, int64_t codes, int64_t e, const Codes& c) {
  uint8_t* m = reinterpret_cast<uint8_t*>(d.exp_avg);
  uint8_t* r = reinterpret_cast<uint8_t*>(d.exp_avg_sq);
  st<u32_at1>(m + e, c.m);
  st<u32_at1>(r + e, c.r);
  if ((threadIdx.x & 15) == 0) {
    m[codes + e / kBlock] = static_cast<uint8_t>(c.me);
    r[codes + e / kBlock] = static_cast<uint8_t>(c.re);
  }
}

// Four values from element e on, `left` of them there (0 to 4; zeros after): whole vectors at any element's alignment.
__device__ __forceinline__ void load_f32(float* v, uint64_t base, int64_t e, int left) {
  const float* p = reinterpret_cast<const float*>(base) + e;
  if (left == 4) {
    const f32x4 a = ld<f32x4_at4>(p);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = j < left ? p[j] : 0.0f;
  }
}
__device__ __forceinline__ void store_f32(uint64_t base, int64_t e, int left, const float* v) {
  float* p = reinterpret_cast<float*>(base) + e;
  if (left == 4) {
    st<f32x4_at4>(p, (f32x4{v[0], v[1], v[2], v[3]}));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < left) p[j] = v[j];
  }
}
__device__ __forceinline__ void load_bf16(float* v, uint64_t base, int64_t e, int left) {
  const uint16_t* p = reinterpret_cast<const uint16_t*>(base) + e;
  if (left == 4) {
    const u32x2 w = ld<u32x2_at2>(p);
    v[0] = bf16_lo(w.x); v[1] = bf16_hi(w.x); v[2] = bf16_lo(w.y); v[3] = bf16_hi(w.y);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = j < left ? bf16_lo(p[j]) : 0.0f;
  }
}
__device__ __forceinline__ void store_bf16(uint64_t base, int64_t e, int left, const float* v) {
  uint16_t* p = reinterpret_cast<uint16_t*>(base) + e;
  const u32x2 w = {pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
  if (left == 4) {
    st<u32x2_at2>(p, w);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < left) p[j] = static_cast<uint16_t>((j < 2 ? w.x : w.y) >> (16 * (j & 1)));
  }
}

// This workgroup's chunk, and the first element of its slice. (A power of two takes a shift for the division's 25
// instructions.)
__device__ __forceinline__ int64_t slice_of(const tm_chunk_t* __restrict__ chunks, uint32_t first_chunk,
                                            uint32_t slices_per_chunk, int64_t chunk_elems, tm_chunk_t& ck) {
  const bool pow2 = (slices_per_chunk & (slices_per_chunk - 1)) == 0;
  const uint32_t local = pow2 ? blockIdx.x >> __builtin_ctz(slices_per_chunk) : blockIdx.x / slices_per_chunk;
  ck = chunks[first_chunk + local];
  return static_cast<int64_t>(ck.chunk) * chunk_elems + static_cast<int64_t>(blockIdx.x - local * slices_per_chunk) * kSlice;
}

// ---------------------------------------------------------------- the step

// What the update needs of a tensor, made once for it (64 bytes, in the workspace).
struct alignas(16) Scal {
  float neg_lrwd, beta1, omb1, beta2, omb2, eps, step_size, inv_bc2s;
  uint32_t key, flags, pad[6];
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
    s.neg_lrwd = s.beta1 = s.omb1 = s.beta2 = s.omb2 = s.eps = s.step_size = s.inv_bc2s = nan;
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
  s.beta1 = static_cast<float>(h.beta1);
  s.omb1 = static_cast<float>(1.0 - h.beta1);
  s.beta2 = static_cast<float>(h.beta2);
  s.omb2 = static_cast<float>(1.0 - h.beta2);
  s.eps = static_cast<float>(h.eps);
  s.step_size = static_cast<float>(h.lr / bc1);
  s.inv_bc2s = static_cast<float>(1.0 / sqrt(bc2));
  s.flags |= h.weight_decay != 0.0 ? kDecay : 0u;
  s.key = mix(static_cast<uint32_t>(fminf(step, 4.0e9f)) + mix(seed_hi + mix(seed_lo)));
  scal[t] = s;
}

// One wave to a slice of 256 elements: 4 a lane, a block of 64 to 16 lanes, whose largest moments meet by DPP moves.
__global__ __launch_bounds__(kWave) void adamw8_update_kernel(const tm_tensor_t* __restrict__ tensors, int64_t n_tensors,
                                                              const tm_chunk_t* __restrict__ chunks, uint32_t first_chunk,
                                                              uint32_t slices_per_chunk, int64_t chunk_elems,
                                                              const Scal* __restrict__ scal,
                                                              const float* __restrict__ coef_p) {
  tm_chunk_t ck;
  const int64_t start = slice_of(chunks, first_chunk, slices_per_chunk, chunk_elems, ck);
  if (ck.tensor >= n_tensors) return;
  const tm_tensor_t d = tensors[ck.tensor];
  if (start >= d.numel) return;  // else the slice's codes are there, whole
  const Scal s = scal[ck.tensor];
  const int64_t e = start + static_cast<int64_t>(threadIdx.x) * 4, codes = held_codes(d.numel);
  const int left = static_cast<int>(max(int64_t(0), min(int64_t(4), d.numel - e)));
  float p[4], g[4], m[4], r[4];
  if (s.flags & kF32) load_f32(g, d.grad, e, left);
  else load_bf16(g, d.grad, e, left);
  load_f32(p, d.master, e, left);
  const Codes was = load_codes(d, codes, e);
  const float coef = (s.flags & kClip) && coef_p ? *coef_p : 1.0f;
  read4(was, m, r);
  uint32_t bits[4];
  const uint32_t z = static_cast<uint32_t>(e) * kHashA + s.key;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float gj = g[j] * coef;
    const float pj = (s.flags & kDecay) ? fmaf(s.neg_lrwd, p[j], p[j]) : p[j];
    m[j] = fmaf(s.beta1, m[j], s.omb1 * gj);
    const float v = fmaf(s.beta2, r[j] * r[j], s.omb2 * gj * gj);
    r[j] = sqrtf(v);
    p[j] = pj - s.step_size * m[j] / fmaf(r[j], s.inv_bc2s, s.eps);
    bits[j] = element_bits(z + j * kHashA);
  }
  const Codes now = hold4(m, r, bits);
  store_f32(d.master, e, left, p);
  store_codes(d, codes, e, now);
  if (s.flags & kOut) store_bf16(d.param_bf16, e, left, p);
}

// ---------------------------------------------------------------- moments as values

// kRead: master = exp_avg's values and grad = the root's, in bf16, or with TM_GRAD_F32 exp_avg's and exp_avg_sq's
// (the root's square) in fp32. Else the fp32 exp_avg and exp_avg_sq there are held, to the nearest.
template <bool kRead>
__global__ __launch_bounds__(kWave) void moments8_kernel(const tm_tensor_t* __restrict__ tensors, int64_t n_tensors,
                                                         const tm_chunk_t* __restrict__ chunks, uint32_t first_chunk,
                                                         uint32_t slices_per_chunk, int64_t chunk_elems) {
  tm_chunk_t ck;
  const int64_t start = slice_of(chunks, first_chunk, slices_per_chunk, chunk_elems, ck);
  if (ck.tensor >= n_tensors) return;
  const tm_tensor_t d = tensors[ck.tensor];
  if (start >= d.numel) return;
  const int64_t e = start + static_cast<int64_t>(threadIdx.x) * 4, codes = held_codes(d.numel);
  const int left = static_cast<int>(max(int64_t(0), min(int64_t(4), d.numel - e)));
  float m[4], r[4];
  if constexpr (kRead) {
    read4(load_codes(d, codes, e), m, r);
    if (d.flags & TM_GRAD_F32) {
#pragma unroll
      for (int j = 0; j < 4; ++j) r[j] *= r[j];
      store_f32(d.master, e, left, m);
      store_f32(d.grad, e, left, r);
    } else {
      store_bf16(d.master, e, left, m);
      store_bf16(d.grad, e, left, r);
    }
  } else {
    load_f32(m, d.master, e, left);
    load_f32(r, d.grad, e, left);
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = sqrtf(r[j]);
    const uint32_t half[4] = {0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u};
    store_codes(d, codes, e, hold4(m, r, half));
  }
}

// kernel(first_chunk, slices_per_chunk, blocks) over a chunk table: launches of less than 2^32 work-items, of
// whole chunks.
template <class F>
int launch_chunks(int64_t n_chunks, int64_t chunk_elems, const char* what, F&& launch) {
  const int64_t spc = chunk_elems / kSlice, per = 0xFFFFFFFFll / kWave / spc;
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
  return launch_chunks(n_chunks, chunk_elems, who, [&](uint32_t first, uint32_t spc, dim3 grid) {
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
  return launch_chunks(n_chunks, chunk_elems, "adamw8_update_kernel", [&](uint32_t first, uint32_t spc, dim3 grid) {
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
