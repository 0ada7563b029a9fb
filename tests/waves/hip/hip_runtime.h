// hip/hip_runtime.h -- for tests only: what the row kernels' sources use of HIP, on the CPU, so that a kernel's every access can be
// checked by the processor. A workgroup runs at a time, each of its work-items on a stack of its own (waves.cpp); a wave's
// lanes go from one collective (ballot, shuffle, readlane) or barrier to the next, the highest lane first. A lane that reads what a
// lower one of its wave then writes therefore reads first, as it does in lockstep.
#pragma once

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>

#define __device__
#define __host__
#define __global__
#define __forceinline__ inline
#define __launch_bounds__(...)
#define __shared__ static

struct dim3 {
  uint32_t x, y, z;
  dim3(uint32_t a = 1, uint32_t b = 1, uint32_t c = 1) : x(a), y(b), z(c) {}
};
extern dim3 blockIdx, gridDim, blockDim;
extern int waves_item;  // the work-item that runs
struct WavesThreadIdx {
  struct {
    operator unsigned() const { return static_cast<unsigned>(waves_item); }
  } x;
};
extern WavesThreadIdx threadIdx;

typedef void* hipStream_t;
typedef int hipError_t;
constexpr hipError_t hipSuccess = 0;
inline hipError_t hipGetLastError() { return hipSuccess; }
inline const char* hipGetErrorString(hipError_t) { return ""; }

void waves_meet();     // all lanes of the wave
void waves_barrier();  // all work-items of the workgroup that have not returned
void waves_launch(dim3 grid, dim3 block, const std::function<void()>& kernel, const char* name);
#define hipLaunchKernelGGL(kernel, grid, block, lds, stream, ...) \
  waves_launch(grid, block, [=] { kernel(__VA_ARGS__); }, #kernel)

inline void __syncthreads() { waves_barrier(); }

extern int64_t waves_slot[1024];
// f(the values of all lanes of the wave)
template <class F>
inline auto waves_exchange(int64_t v, F&& f) {
  waves_slot[waves_item] = v;
  waves_meet();
  const auto r = f(waves_slot + (waves_item & ~63));
  waves_meet();
  return r;
}
inline uint64_t __ballot(bool p) {
  return waves_exchange(p, [](const int64_t* v) {
    uint64_t r = 0;
    for (int i = 0; i < 64; ++i) r |= static_cast<uint64_t>(v[i] != 0) << i;
    return r;
  });
}
inline int __shfl_up(int v, int by, int) {
  const int l = waves_item & 63;
  return static_cast<int>(waves_exchange(v, [&](const int64_t* all) { return all[l >= by ? l - by : l]; }));
}
inline int waves_readlane(int v, int from) {
  if (from < 0 || from > 63) {
    std::printf("readlane of lane %d\n", from);
    std::abort();
  }
  return static_cast<int>(waves_exchange(v, [&](const int64_t* all) { return all[from]; }));
}
#define __builtin_amdgcn_readlane waves_readlane
#define __builtin_amdgcn_readfirstlane(v) waves_readlane(v, 0)

inline int __popcll(unsigned long long v) { return __builtin_popcountll(v); }
inline int __ffsll(unsigned long long v) { return __builtin_ffsll(v); }
inline int atomicAdd(int* p, int v) {
  const int old = *p;
  *p += v;
  return old;
}
inline float __uint_as_float(uint32_t u) {
  float f;
  std::memcpy(&f, &u, 4);
  return f;
}
inline uint32_t __float_as_uint(float f) {
  uint32_t u;
  std::memcpy(&u, &f, 4);
  return u;
}
using std::max;
using std::min;

// What the shared headers name and the kernels that run here do not reach.
typedef float waves_f2 __attribute__((ext_vector_type(2)));
[[noreturn]] inline void waves_absent(const char* what) {
  std::printf("%s is not there on the CPU\n", what);
  std::abort();
}
inline float waves_absent_f(const char* what, ...) { waves_absent(what); }
inline waves_f2 waves_absent_f2(const char* what, ...) { waves_absent(what); }
inline int waves_absent_i(const char* what, ...) { waves_absent(what); }
#define __builtin_amdgcn_rcpf(x) waves_absent_f("rcp", (x))
#define __builtin_amdgcn_exp2f(x) waves_absent_f("exp2", (x))
#define __builtin_amdgcn_fmed3f(a, b, c) waves_absent_f("med3", (a), (b), (c))
#define __builtin_amdgcn_cvt_pk_fp8_f32(a, b, old, high) waves_absent_i("cvt_pk_fp8_f32", (a), (b), (old), (high))
#define __builtin_amdgcn_cvt_pk_f32_fp8(a, high) waves_absent_f2("cvt_pk_f32_fp8", (a), (high))
#define __builtin_amdgcn_update_dpp(old, v, ctrl, rows, banks, bound) waves_absent_i("update_dpp", (v))
