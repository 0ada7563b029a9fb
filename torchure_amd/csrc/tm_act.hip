// tm_act.hip -- gfx950 element-wise kernels around the linear layers' products (tm_linear.hip):
//   quantize_kernel, dequantize_kernel   activations into 8 bits and back (the format: tm_act.h)
//   gate_kernel                          silu(g) u from g and u as held, where no other gradient makes it
//   act_grad_kernel                      dz = dy act'(z) from z as held, with the column sums of dz, and
//   col_sum_kernel                       the bias gradient from those sums
// All are bound by memory: every element is read and written once, 16 bytes a lane.
// Measured (one MI355X): 16,384 x 9728 bf16 into 8 bits 74 us, back 76 (6.3-6.4 TB/s); 8192 x 2560 15 and 14 us; 6001 x 1237
// fp32 10 and 11; silu(g) u of 8192 x 9728 83 us from bf16, 54 from 8 bits (5.8-6.0 TB/s); the slope at 8192 x 9728 83 us
// with its column sums, whose join takes 5.

#include <hip/hip_runtime.h>

#include <stdint.h>

#include <algorithm>

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

template <typename... A>
int act_fail(int code, const char* fmt, A... args) {
  return tm_internal_fail(code, fmt, args...);
}

template <int kV>
struct Int {
  static constexpr int value = kV;
};

// Eight bf16 or fp32 values of a row; `left` of them exist (zeros after). Rows may start at any element: an access of
// 16 bytes need not be aligned to them. (6001 x 1237 values back to fp32, whose rows are odd: 10.9 us so, 25.4 us
// with an access an element.)
template <bool kF32>
struct Raw8 {
  u32x4 w[kF32 ? 2 : 1];
};

// kStream: past the caches (bf16 only; see kStreamBytes).
template <bool kF32, bool kStream = false>
__device__ __forceinline__ Raw8<kF32> get8(const void* base, int64_t at, int left) {
  Raw8<kF32> r = {};
  if constexpr (kF32) {
    const float* p = static_cast<const float*>(base) + at;
    if (left >= 8) {
      r.w[0] = reinterpret_cast<const u32x4_at4*>(p)[0];
      r.w[1] = reinterpret_cast<const u32x4_at4*>(p)[1];
    } else {
#pragma unroll
      for (int e = 0; e < 7; ++e)
        if (e < left) r.w[e / 4][e % 4] = reinterpret_cast<const uint32_t*>(p)[e];
    }
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(base) + at;
    if (left >= 8) {
      const auto* at8 = reinterpret_cast<const u32x4_at2*>(p);
      r.w[0] = kStream ? __builtin_nontemporal_load(at8) : *at8;
    } else {
#pragma unroll
      for (int e = 0; e < 7; ++e)
        if (e < left) r.w[0][e / 2] |= static_cast<uint32_t>(p[e]) << (16 * (e % 2));
    }
  }
  return r;
}

template <bool kF32>
__device__ __forceinline__ void values8(float (&x)[8], const Raw8<kF32>& r) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if constexpr (kF32) x[e] = __uint_as_float(r.w[e / 4][e % 4]);
    else x[e] = e % 2 ? tm_act::bf16_hi(r.w[0][e / 2]) : tm_act::bf16_lo(r.w[0][e / 2]);
  }
}

template <bool kF32, bool kStream = false>
__device__ __forceinline__ void put8(void* base, int64_t at, const float (&x)[8], int left) {
  if constexpr (kF32) {
    float* p = static_cast<float*>(base) + at;
    if (left >= 8) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        reinterpret_cast<u32x4_at4*>(p)[h] = u32x4{__float_as_uint(x[4 * h]), __float_as_uint(x[4 * h + 1]),
                                                   __float_as_uint(x[4 * h + 2]), __float_as_uint(x[4 * h + 3])};
    } else {
#pragma unroll
      for (int e = 0; e < 7; ++e)
        if (e < left) p[e] = x[e];
    }
  } else {
    uint16_t* p = static_cast<uint16_t*>(base) + at;
    const uint32_t w[4] = {pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7])};
    if (left >= 8) {
      auto* at8 = reinterpret_cast<u32x4_at2*>(p);
      const u32x4_at2 v = u32x4{w[0], w[1], w[2], w[3]};
      if constexpr (kStream) __builtin_nontemporal_store(v, at8);
      else *at8 = v;
    } else {
#pragma unroll
      for (int e = 0; e < 7; ++e)
        if (e < left) p[e] = static_cast<uint16_t>(w[e / 2] >> (16 * (e & 1)));
    }
  }
}

// A wave takes 32 rows x 64 columns, two blocks side by side: lane l the columns 8 (l % 8) .. + 7 of rows
// l / 8, + 8, + 16, + 24.
template <bool kF32, bool kStream>
__global__ __launch_bounds__(256) void quantize_kernel(uint8_t* __restrict__ values, uint8_t* __restrict__ exps,
                                                       int64_t ldv, const void* __restrict__ src, int64_t lds,
                                                       int64_t rows, int cols, int wide,
                                                       uint16_t* __restrict__ copy, int64_t ldc) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t band = blockIdx.x / wide;
  const int n0 = (static_cast<int>(blockIdx.x % wide) * 4 + wave) * 64, n = n0 + 8 * (lane & 7);
  if (n0 >= cols) return;
  const int64_t m = band * 32 + (lane >> 3);
  float x[4][8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool in = m + 8 * i < rows;
    values8<kF32>(x[i], get8<kF32, kStream>(src, in ? (m + 8 * i) * lds + n : 0, in ? cols - n : 0));
  }
  // over the block's lanes: l, l ^ 1, l ^ 2, l ^ 8 in a row of 16, and the four rows
  auto over_block = [](uint32_t v) {
    v = max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0xB1, 0xF, 0xF, true)));
    v = max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x4E, 0xF, 0xF, true)));
    v = max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x128, 0xF, 0xF, true)));
#pragma unroll
    for (int d : {16, 32}) v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), d)));
    return v;
  };
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) most = max(most, tm_act::largest<8>(x[i]));
  most = over_block(most);
  auto encode = [&](auto any) {
    constexpr bool kAny = decltype(any)::value != 0;
    const int e2 = tm_act::block_exponent(most);
    const float inv = tm_act::two_to(-e2);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (m + 8 * i >= rows) continue;
      if (n < ldv) {
        const u32x2 w = {tm_act::encode4<kAny>(x[i][0], x[i][1], x[i][2], x[i][3], inv),
                         tm_act::encode4<kAny>(x[i][4], x[i][5], x[i][6], x[i][7], inv)};
        *reinterpret_cast<u32x2*>(values + (m + 8 * i) * ldv + n) = w;
      }
      if (copy && n < ldc) put8<false>(copy, (m + 8 * i) * ldc + n, x[i], 8);
    }
    const int block = (n0 >> 5) + ((lane >> 2) & 1);
    if ((lane & ~4) == 0 && block * 32 < cols)
      exps[band * ((cols + 31) / 32) + block] = static_cast<uint8_t>(e2 + 127);
  };
  if (__builtin_amdgcn_ballot_w64(most >= tm_act::kPlainMost) == 0) {
    encode(Int<0>{});
  } else {  // some block with an infinity or values next to the type's largest
    most = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) most = max(most, tm_act::largest_finite<8>(x[i]));
    most = over_block(most);
    encode(Int<1>{});
  }
}

template <bool kF32, bool kStream>
__global__ __launch_bounds__(256) void dequantize_kernel(void* __restrict__ dst, int64_t ldd,
                                                         const uint8_t* __restrict__ values,
                                                         const uint8_t* __restrict__ exps, int64_t ldv, int64_t rows,
                                                         int cols, int wide) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t band = blockIdx.x / wide;
  const int n0 = (static_cast<int>(blockIdx.x % wide) * 4 + wave) * 64, n = n0 + 8 * (lane & 7);
  if (n >= cols) return;
  const int64_t m = band * 32 + (lane >> 3);
  const float scale = tm_act::two_to(static_cast<int>(exps[band * ((cols + 31) / 32) + (n >> 5)]) - 127);
  u32x2 w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (m + 8 * i < rows) w[i] = *reinterpret_cast<const u32x2*>(values + (m + 8 * i) * ldv + n);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (m + 8 * i >= rows) continue;
    const f32x4 a = tm_act::decode4(w[i].x, scale), b = tm_act::decode4(w[i].y, scale);
    const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    put8<kF32, kStream>(dst, (m + 8 * i) * ldd + n, x, cols - n);
  }
}

// silu(g) u, a wave's elements as above, each by the operations of the gate's gradient (tm_linear.hip), so with its bits.
// Columns from cols to the next multiple of 8 are held as zeros.
template <bool kE4m3>
__global__ __launch_bounds__(256) void gate_kernel(uint16_t* __restrict__ dst, int64_t ldd,
                                                   const uint8_t* __restrict__ g, const uint8_t* __restrict__ u,
                                                   const uint8_t* __restrict__ g_exps,
                                                   const uint8_t* __restrict__ u_exps, int64_t ldz, int64_t rows,
                                                   int cols, int wide) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t band = blockIdx.x / wide;
  const int n = (static_cast<int>(blockIdx.x % wide) * 4 + wave) * 64 + 8 * (lane & 7);
  if (n >= cols) return;
  const int64_t m = band * 32 + (lane >> 3);
  u32x4 a[4], b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (m + 8 * i >= rows) continue;
    const int64_t at = (m + 8 * i) * ldz + n;
    if constexpr (kE4m3) {
      const u32x2 x = *reinterpret_cast<const u32x2*>(g + at), y = *reinterpret_cast<const u32x2*>(u + at);
      a[i] = u32x4{x.x, x.y, 0, 0};
      b[i] = u32x4{y.x, y.y, 0, 0};
    } else {
      a[i] = *reinterpret_cast<const u32x4*>(g + 2 * at);
      b[i] = *reinterpret_cast<const u32x4*>(u + 2 * at);
    }
  }
  float sg = 1.0f, su = 1.0f;
  if constexpr (kE4m3) {
    const int64_t at = band * ((cols + 31) / 32) + (n >> 5);
    sg = tm_act::two_to(static_cast<int>(g_exps[at]) - 127);
    su = tm_act::two_to(static_cast<int>(u_exps[at]) - 127);
  }
  auto values = [](float (&x)[8], const u32x4& w, float scale) {
    if constexpr (kE4m3) {
      const f32x4 lo = tm_act::decode4(w.x, scale), hi = tm_act::decode4(w.y, scale);
      x[0] = lo.x; x[1] = lo.y; x[2] = lo.z; x[3] = lo.w;
      x[4] = hi.x; x[5] = hi.y; x[6] = hi.z; x[7] = hi.w;
    } else {
      values8<false>(x, Raw8<false>{{w}});
    }
  };
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (m + 8 * i >= rows) continue;
    float z[8], h[8];
    values(z, a[i], sg);
    values(h, b[i], su);
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] *= z[e] * tm_act::sigmoid(z[e]);
    put8<false>(dst, (m + 8 * i) * ldd + n, h, 8);
  }
}

// Rows of a workgroup, and of one partial column sum where those are made. (8192 x 1024 fp32 dy cast to bf16: 19.8 us
// with 128 rows, whose 256 workgroups leave a CU with four waves.)
constexpr int kBandRows = 64, kPlainRows = 32;

// A workgroup takes `band_rows` rows x 256 columns: thread t the columns 8 (t % 32) .. + 7 of rows t / 32, + 8, ...,
// four rows' loads at once, without branches (where the ways of reading z met, each row's loads were waited for:
// 8192 x 9728 bf16 dy and 8-bit z, silu, 103 us then, 83 us now, 4.8 TB/s).
template <bool kF32, int kAct, bool kE4m3>
__global__ __launch_bounds__(256) void act_grad_kernel(uint16_t* __restrict__ dz, int64_t lddz,
                                                       float* __restrict__ sums, const void* __restrict__ dy,
                                                       int64_t ldy, const uint8_t* __restrict__ z,
                                                       const uint8_t* __restrict__ exps, int64_t ldz, int64_t rows,
                                                       int cols, int wide, int band_rows) {
  const int t = threadIdx.x;
  const int64_t band = blockIdx.x / wide;
  const int n = static_cast<int>(blockIdx.x % wide) * 256 + 8 * (t & 31);
  const int64_t m_end = min(rows, (band + 1) * band_rows);
  const int blocks = (cols + 31) / 32;
  float total[8] = {};
  if (n < cols) {
    for (int64_t m0 = band * band_rows; m0 < m_end; m0 += 32) {
      Raw8<kF32> d4[4];
      Raw8<false> z4[4];
      uint32_t exp = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t m = min(m0 + (t >> 5) + 8 * i, m_end - 1);
        d4[i] = get8<kF32>(dy, m * ldy + n, cols - n);
        if constexpr (kAct != TM_ACT_NONE && kE4m3) {
          const u32x2 w = *reinterpret_cast<const u32x2*>(z + m * ldz + n);
          z4[i].w[0] = u32x4{w.x, w.y, 0, 0};
        } else if constexpr (kAct != TM_ACT_NONE) {
          z4[i].w[0] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(z) + m * ldz + n);
        }
      }
      if constexpr (kAct != TM_ACT_NONE && kE4m3) exp = exps[(m0 >> 5) * blocks + (n >> 5)];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t m = m0 + (t >> 5) + 8 * i;
        if (m >= m_end) break;
        float d[8];
        values8<kF32>(d, d4[i]);
        if constexpr (kAct != TM_ACT_NONE) {
          float x[8];
          if constexpr (kE4m3) {
            const float scale = tm_act::two_to(static_cast<int>(exp) - 127);
            const f32x4 a = tm_act::decode4(z4[i].w[0].x, scale), b = tm_act::decode4(z4[i].w[0].y, scale);
            x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
            x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
          } else {
            values8<false>(x, z4[i]);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) d[e] = n + e < cols ? d[e] * tm_act::act1_grad(kAct, x[e]) : 0.0f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) total[e] += d[e];
        if (dz) put8<false>(dz, m * lddz + n, d, 8);
      }
    }
  } else if (dz && n < lddz) {  // whole groups of padding
    const float none[8] = {};
    for (int64_t m = band * band_rows + (t >> 5); m < m_end; m += 8) put8<false>(dz, m * lddz + n, none, 8);
  }
  if (!sums) return;
  __shared__ float part[8][256];
#pragma unroll
  for (int e = 0; e < 8; ++e) part[t >> 5][8 * (t & 31) + e] = total[e];
  __syncthreads();
  const int c = static_cast<int>(blockIdx.x % wide) * 256 + t;
  if (c >= cols) return;
  float sum = part[0][t];
#pragma unroll
  for (int r = 1; r < 8; ++r) sum += part[r][t];
  sums[band * cols + c] = sum;
}

// A column's partial sums, a quarter of the bands by each of a workgroup's waves, then the quarters, in order.
__global__ __launch_bounds__(256) void col_sum_kernel(void* __restrict__ out, int f32, const float* __restrict__ sums,
                                                      int64_t bands, int cols) {
  __shared__ float part[4][64];
  const int c = static_cast<int>(blockIdx.x) * 64 + (threadIdx.x & 63), w = threadIdx.x >> 6;
  const int64_t per = (bands + 3) / 4, from = w * per, to = min(bands, from + per);
  float sum = 0.0f;
  if (c < cols)
#pragma unroll 8
    for (int64_t b = from; b < to; ++b) sum += sums[b * cols + c];
  part[w][threadIdx.x & 63] = sum;
  __syncthreads();
  if (w || c >= cols) return;
  sum = ((part[0][threadIdx.x] + part[1][threadIdx.x]) + part[2][threadIdx.x]) + part[3][threadIdx.x];
  if (f32) static_cast<float*>(out)[c] = sum;
  else static_cast<uint16_t*>(out)[c] = static_cast<uint16_t>(pack_bf16(sum, sum));
}

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// bf16 matrices of more bytes than this go past the caches, which then keep the 8-bit values, unless the caller says that
// they are read next. (Into 8 bits and back, us past / through them: 320 MB 150 / 180, 192 MB 93 / 115, 128 MB 65 / 70,
// but 96 MB 50 / 47, 64 MB 34 / 33; fp32, whose lanes have 32 bytes each, 202 / 173 at 320 MB. Into 8 bits and through a
// product of 128 columns, which finds part of the matrix in the caches: 175 MB 99 / 94, back and through the weight's
// gradient 102 / 91; of 1024 columns, 169 MB, 195 / 190 and 197 / 197; at 320 MB no difference.)
constexpr int64_t kStreamBytes = int64_t(160) << 20;

// A launch has less than 2^32 work-items, 256 a workgroup.
constexpr int64_t kMaxRows = int64_t(1) << 30, kMaxCols = int64_t(1) << 30, kMaxGroups = (int64_t(1) << 24) - 1;

int check_shape(const char* who, int64_t rows, int64_t cols, int64_t groups) {
  if (rows < 0 || cols < 0 || rows > kMaxRows || cols > kMaxCols || groups > kMaxGroups)
    return act_fail(TM_EINVAL, "%s: %lld rows of %lld are negative or too large", who, (long long)rows, (long long)cols);
  return TM_OK;
}

int launched(const char* who) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? TM_OK : act_fail(TM_ELAUNCH, "%s: launch failed: %s", who, hipGetErrorString(e));
}

}  // namespace

extern "C" {

int tm_quantize_e4m3(uint8_t* d_values, uint8_t* d_exponents, int64_t ldv, const void* d_src, int src_f32, int64_t lds,
                     int64_t rows, int64_t cols, uint16_t* d_copy, int64_t ldc, void* stream) {
  const char* who = "tm_quantize_e4m3";
  if (src_f32 & ~(1 | TM_READ_NEXT)) return act_fail(TM_EINVAL, "%s: unknown flags %d", who, src_f32);
  const bool f32 = src_f32 & 1;
  const int64_t wide = ceil_div(cols, 256), groups = rows > 0 && cols > 0 ? ceil_div(rows, 32) * wide : 0;
  if (const int rc = check_shape(who, rows, cols, groups)) return rc;
  if (groups == 0) return TM_OK;
  if (!d_values || !d_exponents || !d_src) return act_fail(TM_EINVAL, "%s: null pointer", who);
  if (ldv != ceil_div(cols, 32) * 32 || !aligned(d_values, 16) || lds < cols || !aligned(d_src, f32 ? 4 : 2))
    return act_fail(TM_EINVAL, "%s: values (rows %lld apart) need rows of the next multiple of 32 to %lld, 16-byte "
                    "aligned; source rows are %lld apart", who, (long long)ldv, (long long)cols, (long long)lds);
  if (d_copy && (ldc != ceil_div(cols, 8) * 8 || !aligned(d_copy, 16)))
    return act_fail(TM_EINVAL, "%s: copy rows %lld apart for %lld columns: the next multiple of 8, 16-byte aligned", who,
                    (long long)ldc, (long long)cols);
  const bool past = !f32 && !(src_f32 & TM_READ_NEXT) && rows * cols * 2 > kStreamBytes;
  const dim3 grid(static_cast<uint32_t>(groups));
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto launch = [&](auto kind, auto stream8) {
    hipLaunchKernelGGL((quantize_kernel<decltype(kind)::value != 0, decltype(stream8)::value != 0>), grid, dim3(256), 0, s,
                       d_values, d_exponents, ldv, d_src, lds, rows, static_cast<int>(cols), static_cast<int>(wide),
                       d_copy, ldc);
  };
  if (f32) launch(Int<1>{}, Int<0>{});
  else if (past) launch(Int<0>{}, Int<1>{});
  else launch(Int<0>{}, Int<0>{});
  return launched(who);
}

int tm_dequantize_e4m3(void* d_dst, int dst_f32, int64_t ldd, const uint8_t* d_values, const uint8_t* d_exponents,
                       int64_t ldv, int64_t rows, int64_t cols, void* stream) {
  const char* who = "tm_dequantize_e4m3";
  if (dst_f32 & ~(1 | TM_READ_NEXT)) return act_fail(TM_EINVAL, "%s: unknown flags %d", who, dst_f32);
  const bool f32 = dst_f32 & 1;
  const int64_t wide = ceil_div(cols, 256), groups = rows > 0 && cols > 0 ? ceil_div(rows, 32) * wide : 0;
  if (const int rc = check_shape(who, rows, cols, groups)) return rc;
  if (groups == 0) return TM_OK;
  if (!d_values || !d_exponents || !d_dst) return act_fail(TM_EINVAL, "%s: null pointer", who);
  if (ldv != ceil_div(cols, 32) * 32 || !aligned(d_values, 16) || ldd < cols || !aligned(d_dst, f32 ? 4 : 2))
    return act_fail(TM_EINVAL, "%s: values (rows %lld apart) need rows of the next multiple of 32 to %lld, 16-byte "
                    "aligned; output rows are %lld apart", who, (long long)ldv, (long long)cols, (long long)ldd);
  const bool past = !f32 && !(dst_f32 & TM_READ_NEXT) && rows * cols * 2 > kStreamBytes;
  const dim3 grid(static_cast<uint32_t>(groups));
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto launch = [&](auto kind, auto stream8) {
    hipLaunchKernelGGL((dequantize_kernel<decltype(kind)::value != 0, decltype(stream8)::value != 0>), grid, dim3(256), 0, s,
                       d_dst, ldd, d_values, d_exponents, ldv, rows, static_cast<int>(cols), static_cast<int>(wide));
  };
  if (f32) launch(Int<1>{}, Int<0>{});
  else if (past) launch(Int<0>{}, Int<1>{});
  else launch(Int<0>{}, Int<0>{});
  return launched(who);
}

int tm_held_gate(uint16_t* d_dst, int64_t ldd, const void* d_g, const void* d_u, const uint8_t* d_g_exponents,
                 const uint8_t* d_u_exponents, int64_t ldz, int held, int64_t rows, int64_t cols, void* stream) {
  const char* who = "tm_held_gate";
  const int64_t wide = ceil_div(cols, 256), groups = rows > 0 && cols > 0 ? ceil_div(rows, 32) * wide : 0;
  if (const int rc = check_shape(who, rows, cols, groups)) return rc;
  if (groups == 0) return TM_OK;
  if (!d_dst || !d_g || !d_u || (held == TM_HELD_E4M3 && (!d_g_exponents || !d_u_exponents)))
    return act_fail(TM_EINVAL, "%s: null pointer", who);
  if (ldd % 8 || ldd < cols || !aligned(d_dst, 16) || !aligned(d_g, 16) || !aligned(d_u, 16))
    return act_fail(TM_EINVAL, "%s: output rows %lld apart for %lld columns: a multiple of 8; all 16-byte aligned", who,
                    (long long)ldd, (long long)cols);
  if (held == TM_HELD_BF16 ? ldz % 8 || ldz < cols : held != TM_HELD_E4M3 || ldz != ceil_div(cols, 32) * 32)
    return act_fail(TM_EINVAL, "%s: held as %d in rows %lld apart for %lld columns", who, held, (long long)ldz,
                    (long long)cols);
  const dim3 grid(static_cast<uint32_t>(groups));
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto launch = [&](auto e4m3) {
    hipLaunchKernelGGL((gate_kernel<decltype(e4m3)::value != 0>), grid, dim3(256), 0, s, d_dst, ldd,
                       static_cast<const uint8_t*>(d_g), static_cast<const uint8_t*>(d_u), d_g_exponents, d_u_exponents,
                       ldz, rows, static_cast<int>(cols), static_cast<int>(wide));
  };
  if (held == TM_HELD_E4M3) launch(Int<1>{});
  else launch(Int<0>{});
  return launched(who);
}

size_t tm_act_grad_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  return static_cast<size_t>(ceil_div(rows, kBandRows)) * cols * sizeof(float);
}

int tm_act_grad(uint16_t* d_dz, int64_t lddz, void* d_bias, int bias_f32, const void* d_dy, int dy_f32, int64_t ldy,
                const void* d_z, const uint8_t* d_exponents, int64_t ldz, int held, int act, int64_t rows, int64_t cols,
                void* d_ws, size_t ws_bytes, void* stream) {
  const char* who = "tm_act_grad";
  const int64_t wide = ceil_div(d_dz && lddz > cols ? lddz : cols, 256);
  const int band_rows = d_bias ? kBandRows : kPlainRows;
  const int64_t bands = rows > 0 ? ceil_div(rows, band_rows) : 0;
  if (const int rc = check_shape(who, rows, cols, std::max<int64_t>(bands * wide, d_bias ? ceil_div(cols, 64) : 0))) return rc;
  if (rows == 0 || cols == 0) return act_fail(TM_EINVAL, "%s: no elements", who);
  if (!d_dy || (!d_dz && !d_bias)) return act_fail(TM_EINVAL, "%s: null pointer", who);
  if (act < 0 || act > TM_ACT_GELU_TANH) return act_fail(TM_EINVAL, "%s: unknown activation %d", who, act);
  if (ldy < cols || !aligned(d_dy, dy_f32 ? 4 : 2))
    return act_fail(TM_EINVAL, "%s: dy rows %lld apart for %lld columns", who, (long long)ldy, (long long)cols);
  if (d_dz && (lddz % 8 || lddz < cols || lddz - cols >= 256 || !aligned(d_dz, 16)))
    return act_fail(TM_EINVAL, "%s: dz rows %lld apart for %lld columns, 16-byte aligned", who, (long long)lddz,
                    (long long)cols);
  if (act != TM_ACT_NONE) {
    if (!d_z || !aligned(d_z, 16) || (held == TM_HELD_E4M3 && !d_exponents))
      return act_fail(TM_EINVAL, "%s: z must be 16-byte aligned, not null", who);
    if (held == TM_HELD_BF16 ? ldz % 8 || ldz < cols : held != TM_HELD_E4M3 || ldz != ceil_div(cols, 32) * 32)
      return act_fail(TM_EINVAL, "%s: z held as %d in rows %lld apart for %lld columns", who, held, (long long)ldz,
                      (long long)cols);
  }
  const size_t need = d_bias ? tm_act_grad_workspace_bytes(rows, cols) : 0;
  if (need && (!d_ws || ws_bytes < need || !aligned(d_ws, 4)))
    return act_fail(TM_EINVAL, "%s: workspace of %zu bytes, %zu needed", who, ws_bytes, need);
  float* sums = d_bias ? static_cast<float*>(d_ws) : nullptr;
  const dim3 grid(static_cast<uint32_t>(bands * wide));
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto launch = [&](auto f32, auto a, auto e4m3) {
    hipLaunchKernelGGL((act_grad_kernel<decltype(f32)::value != 0, decltype(a)::value, decltype(e4m3)::value != 0>), grid,
                       dim3(256), 0, s, d_dz, lddz, sums, d_dy, ldy, static_cast<const uint8_t*>(d_z), d_exponents, ldz,
                       rows, static_cast<int>(cols), static_cast<int>(wide), band_rows);
  };
  auto by_held = [&](auto f32, auto a) {
    if (held == TM_HELD_E4M3) launch(f32, a, Int<1>{});
    else launch(f32, a, Int<0>{});
  };
  auto by_act = [&](auto f32) {
    switch (act) {
      case TM_ACT_NONE: return launch(f32, Int<TM_ACT_NONE>{}, Int<0>{});
      case TM_ACT_RELU: return by_held(f32, Int<TM_ACT_RELU>{});
      case TM_ACT_SILU: return by_held(f32, Int<TM_ACT_SILU>{});
      case TM_ACT_GELU: return by_held(f32, Int<TM_ACT_GELU>{});
      default: return by_held(f32, Int<TM_ACT_GELU_TANH>{});
    }
  };
  if (dy_f32) by_act(Int<1>{});
  else by_act(Int<0>{});
  if (const int rc = launched(who)) return rc;
  if (!d_bias) return TM_OK;
  hipLaunchKernelGGL(col_sum_kernel, dim3(static_cast<uint32_t>(ceil_div(cols, 64))), dim3(256), 0, s, d_bias, bias_f32,
                     sums, bands, static_cast<int>(cols));
  return launched(who);
}

}  // extern "C"
