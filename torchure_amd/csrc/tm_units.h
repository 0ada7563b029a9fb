// tm_units.h -- units of 4 or 8 neighbouring elements of a bf16 or fp32 row, as the row kernels read and write them: one
// access of 8 or 16 bytes at any element's alignment, element by element at a row's end.
#ifndef TM_UNITS_H
#define TM_UNITS_H

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "tm_act.h"

namespace tm_units {

using tm_act::u32x2;
using tm_act::u32x4;
using tm_act::u32x4_at2;
using tm_act::u32x4_at4;
typedef u32x2 u32x2_at2 __attribute__((aligned(2)));

// A unit as it was read.
template <bool kF32, int kU>
struct Raw {
  static_assert(!kF32 || kU == 4, "at most 16 bytes");
  uint32_t w[kF32 ? kU : kU / 2];
};

// `left` of its elements exist; zeros after. kStream: past the caches.
template <bool kF32, int kU, bool kStream = false>
__device__ __forceinline__ Raw<kF32, kU> read(const void* base, int64_t at, int left) {
  Raw<kF32, kU> r = {};
  if constexpr (kF32) {
    const uint32_t* p = static_cast<const uint32_t*>(base) + at;
    if (left >= 4) {
      const auto* q = reinterpret_cast<const u32x4_at4*>(p);
      const u32x4 a = kStream ? __builtin_nontemporal_load(q) : *q;
#pragma unroll
      for (int i = 0; i < 4; ++i) r.w[i] = a[i];
    } else {
#pragma unroll
      for (int i = 0; i < 3; ++i)
        if (i < left) r.w[i] = p[i];
    }
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(base) + at;
    if (left >= kU) {
      if constexpr (kU == 8) {
        const auto* q = reinterpret_cast<const u32x4_at2*>(p);
        const u32x4 a = kStream ? __builtin_nontemporal_load(q) : *q;
#pragma unroll
        for (int i = 0; i < 4; ++i) r.w[i] = a[i];
      } else {
        const auto* q = reinterpret_cast<const u32x2_at2*>(p);
        const u32x2 a = kStream ? __builtin_nontemporal_load(q) : *q;
        r.w[0] = a.x;
        r.w[1] = a.y;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kU - 1; ++i)
        if (i < left) r.w[i / 2] |= static_cast<uint32_t>(p[i]) << (16 * (i & 1));
    }
  }
  return r;
}

template <bool kF32, int kU>
__device__ __forceinline__ void values(float (&v)[kU], const Raw<kF32, kU>& r) {
#pragma unroll
  for (int i = 0; i < kU; ++i) {
    if constexpr (kF32) v[i] = __uint_as_float(r.w[i]);
    else v[i] = i % 2 ? tm_act::bf16_hi(r.w[i / 2]) : tm_act::bf16_lo(r.w[i / 2]);
  }
}

template <bool kF32, int kU, bool kStream = false>
__device__ __forceinline__ void get(float (&v)[kU], const void* base, int64_t at, int left) {
  values(v, read<kF32, kU, kStream>(base, at, left));
}

template <bool kF32, int kU, bool kStream = false>
__device__ __forceinline__ void put(void* base, int64_t at, const float (&v)[kU], int left) {
  if constexpr (kF32) {
    float* p = static_cast<float*>(base) + at;
    if (left >= 4) {
      auto* q = reinterpret_cast<u32x4_at4*>(p);
      const u32x4_at4 a = u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
      if constexpr (kStream) __builtin_nontemporal_store(a, q);
      else *q = a;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < left) p[i] = v[i];
    }
  } else {
    uint16_t* p = static_cast<uint16_t*>(base) + at;
    uint32_t w[kU / 2];
#pragma unroll
    for (int i = 0; i < kU / 2; ++i) w[i] = tm_act::pack_bf16(v[2 * i], v[2 * i + 1]);
    if (left >= kU) {
      if constexpr (kU == 8) {
        auto* q = reinterpret_cast<u32x4_at2*>(p);
        const u32x4_at2 a = u32x4{w[0], w[1], w[2], w[3]};
        if constexpr (kStream) __builtin_nontemporal_store(a, q);
        else *q = a;
      } else {
        auto* q = reinterpret_cast<u32x2_at2*>(p);
        const u32x2_at2 a = u32x2{w[0], w[1]};
        if constexpr (kStream) __builtin_nontemporal_store(a, q);
        else *q = a;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kU; ++i)
        if (i < left) p[i] = static_cast<uint16_t>(w[i / 2] >> (16 * (i & 1)));
    }
  }
}

}  // namespace tm_units

#endif
