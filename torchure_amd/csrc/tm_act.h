// tm_act.h -- device arithmetic shared by the linear layers' translation units: the activations with
// their derivatives, and the 8-bit format activations are held in between forward and backward.
//
// The 8-bit format: e4m3 values (4 exponent bits, 3 of mantissa, largest 448, no infinities) and one
// exponent byte e + 127 for each block of 32 rows x 32 columns. e is the least exponent with which
// the block's largest finite magnitude is at most 448 2^e, clamped to [-117, 119]. A value is off by at most 2^-4
// of itself where it is at least 2^-6 2^e (2^-13.8 of the block's largest, or less), else by at most 2^-10 2^e;
// every held value, v 2^e, is a normal bf16 number or zero: reading back rounds nothing. (e4m3 is itself a floating format:
// a block's scale sets its range, not its step. A square block keeps that scale the same along rows
// and columns, so a product may contract either, and costs 1 byte in 1024.) Values past 448 2^119
// (over 2.98e38) are held as that, infinities and NaN as NaN.
#ifndef TM_ACT_H
#define TM_ACT_H

#include <hip/hip_runtime.h>

#include <stdint.h>

namespace tm_act {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_at2 __attribute__((aligned(2)));  // where rows start at any bf16, at any fp32
typedef u32x4 u32x4_at4 __attribute__((aligned(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

enum Act { kNone = 0, kRelu = 1, kSilu = 2, kGelu = 3, kGeluTanh = 4 };

// Two floats -> packed bf16, round to nearest even (v_cvt_pk_bf16_f32).
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const bf16x2 h = __builtin_convertvector(f32x2{a, b}, bf16x2);
  return __builtin_bit_cast(uint32_t, h);
}
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

// 1 / (1 + exp(-z)): exp2 and the reciprocal are each within an ulp, the exponent's rounding adds
// |z| 2^-24 relative. exp2 past the range gives inf, whose reciprocal is the limit 0.
__device__ __forceinline__ float sigmoid(float z) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.4426950408889634f));
}

constexpr float kGeluC = 1.5957691216057308f;  // 2 sqrt(2 / pi): (1 + tanh u) / 2 = sigmoid(2 u)

// The normal distribution function and exp(-z^2 / 2): Abramowitz and Stegun's formula 7.1.26 for the
// error function of |z| / sqrt 2, at most 1.5e-7 off (half of that here), taken on the tail's side.
__device__ __forceinline__ float normal_cdf(float z, float& bell) {
  const float t = __builtin_amdgcn_rcpf(1.0f + 0.23164190f * fabsf(z));  // 0.3275911 / sqrt 2
  bell = __builtin_amdgcn_exp2f(z * z * -0.72134752044448170f);
  const float poly =
      t * (0.127414796f + t * (-0.142248368f + t * (0.7107068705f + t * (-0.7265760135f + t * 0.5307027145f))));
  const float tail = poly * bell;
  return z < 0.0f ? tail : 1.0f - tail;
}

__device__ __forceinline__ float act1(int act, float z) {
  float bell;
  switch (act) {
    case kRelu: return z < 0.0f ? 0.0f : z;  // NaN stays
    case kSilu: return z * sigmoid(z);
    case kGelu: return z * normal_cdf(z, bell);
    case kGeluTanh: return z * sigmoid(kGeluC * z * (1.0f + 0.044715f * z * z));
    default: return z;
  }
}

__device__ __forceinline__ float silu_grad(float z, float s) { return s * (1.0f + z * (1.0f - s)); }

__device__ __forceinline__ float act1_grad(int act, float z) {
  float bell;
  switch (act) {
    case kRelu: return z > 0.0f ? 1.0f : 0.0f;
    case kSilu: return silu_grad(z, sigmoid(z));
    case kGelu: {
      const float cdf = normal_cdf(z, bell);
      return cdf + z * 0.39894228040143268f * bell;
    }
    case kGeluTanh: {
      // s (1 - s) is zero long before the square's limit
      const float z2 = fminf(z * z, 1e6f), s = sigmoid(kGeluC * z * (1.0f + 0.044715f * z2));
      return s + z * s * (1.0f - s) * kGeluC * (1.0f + 0.134145f * z2);
    }
    default: return 1.0f;
  }
}

// ---------------------------------------------------------------- e4m3 with a block exponent

// |x| as bits where x is finite, else 0: unsigned integers of the same order.
__device__ __forceinline__ uint32_t finite_bits(float x) {
  const uint32_t u = __float_as_uint(x) & 0x7FFFFFFFu;
  return u < 0x7F800000u ? u : 0u;
}

// The block's exponent from its largest finite magnitude's bits: m 2^E, 1 <= m < 2, needs E - 8
// (448 = 1.75 2^8), one more if m > 1.75.
__device__ __forceinline__ int block_exponent(uint32_t most) {
  const int e = static_cast<int>(most >> 23) - 135 + ((most & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return min(max(e, -117), 119);
}
__device__ __forceinline__ float two_to(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// Four values times `inv` (2^-e) -> four e4m3 bytes, round to nearest even. kAny: any values; else none past the
// range (NaN becomes NaN).
__device__ __forceinline__ float e4m3_range(float x, float inv) {
  const float c = __builtin_amdgcn_fmed3f(x * inv, -448.0f, 448.0f);
  return finite_bits(x) != 0u || x == 0.0f ? c : __uint_as_float(0x7FC00000u);
}
template <bool kAny>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d, float inv) {
  uint32_t w = 0;
  if constexpr (kAny) {
    w = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_range(a, inv), e4m3_range(b, inv), w, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_range(c, inv), e4m3_range(d, inv), w, true);
  } else {
    w = __builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, w, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, w, true);
  }
  return w;
}

// The largest over the 16 lanes of a row, in each of them. (DPP moves: no LDS.)
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
  v = max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x121, 0xF, 0xF, true)));
  v = max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x122, 0xF, 0xF, true)));
  v = max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x124, 0xF, 0xF, true)));
  return max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x128, 0xF, 0xF, true)));
}
// ... over the wave.
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  v = row_max(v);
  const uint32_t a = max(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 0)),
                         static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 16)));
  const uint32_t b = max(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 32)),
                         static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 48)));
  return max(a, b);
}

// Past this a block's values are looked at one by one (the clamped exponent, infinities); below, the largest
// magnitude that is no NaN is the largest finite one, and times 2^-e nothing is past 448.
constexpr uint32_t kPlainMost = 0x7F600000u;  // 1.75 2^127
// The largest magnitude of n values as bits, NaN left out.
template <int n>
__device__ __forceinline__ uint32_t largest(const float* x) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < n; ++i) m = fmaxf(m, fabsf(x[i]));
  return __float_as_uint(m);
}
template <int n>
__device__ __forceinline__ uint32_t largest_finite(const float* x) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < n; ++i) m = max(m, finite_bits(x[i]));
  return m;
}

// Four e4m3 bytes times `scale` (2^e), exact.
__device__ __forceinline__ f32x4 decode4(uint32_t w, float scale) {
  const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  return f32x4{lo.x * scale, lo.y * scale, hi.x * scale, hi.y * scale};
}

}  // namespace tm_act

#endif
