// tm_norm.hip -- gfx950 kernels of layer norm and RMS norm over a matrix's rows, forward and backward.
//
//   forward    xhat = (x - mean) rstd,  rstd = 1 / sqrt(mean((x - mean)^2) + eps),  y = xhat w + b   (RMS: mean = 0)
//   backward   g = dy w,  dx = rstd (g - mean(g xhat) xhat - mean(g)),  dw = sum over rows of dy xhat,  db = of dy
//              (RMS: without mean(g) and db)
//
// Both are bound by memory: x in, y out; x and dy in, dx out. A row stays in the registers of the lanes that it is dealt to, between
// its loads and its results, so the statistics take two passes over registers (the sum of squared distances from the mean, not of
// squares) and no second read. A row has 8 to 64 lanes of a wave, or whole workgroups of 4 or 8 waves, by its length; lanes
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

template <typename... A>
int fail(int code, const char* fmt, A... args) {
  return tm_internal_fail(code, fmt, args...);
}

constexpr int kWave = 64;
constexpr int kCus = 256;

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

// The sum over a row: its kLanes lanes, or the workgroup's. `room`: 2 x 8 floats of LDS used in turn: a wave writes one half
// again only after a barrier that every wave reaches when it has read it.
template <int kLanes>
struct RowSum {
  float* room;
  int turn = 0;
  __device__ __forceinline__ float operator()(float v) {
    if constexpr (kLanes <= kWave) {
      return group_sum<kLanes>(v);
    } else {
      constexpr int kWaves = kLanes / kWave;
      v = group_sum<kWave>(v);
      float* r = room + 8 * turn;
      turn ^= 1;
      if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = v;
      __syncthreads();
      float s = r[0];
#pragma unroll
      for (int i = 1; i < kWaves; ++i) s += r[i];
      return s;
    }
  }
};

// A kernel's shape: kLanes lanes to a row, kVec units of kU elements to a lane; kThreads to a workgroup.
template <int kLanes_, int kVec_, int kU_>
struct Shape {
  static constexpr int kLanes = kLanes_, kVec = kVec_, kU = kU_;
  static constexpr int kThreads = kLanes <= kWave ? 256 : kLanes;
  static constexpr int kRows = kThreads / kLanes;  // rows of a workgroup at a time
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

template <int kU>
__device__ __forceinline__ void param(float (&v)[kU], const void* p, int f32, int at, int cols, float otherwise) {
#pragma unroll
  for (int i = 0; i < kU; ++i) {
    float a = otherwise;
    if (p && at + i < cols)
      a = f32 ? static_cast<const float*>(p)[at + i] : bf16_lo(static_cast<const uint16_t*>(p)[at + i]);
    v[i] = a;
  }
}

template <class S, bool kX32, bool kY32, bool kLayer>
__global__ __launch_bounds__(S::kThreads) void norm_forward_kernel(Forward a) {
  __shared__ float room[16];
  RowSum<S::kLanes> row_sum{room};
  const int l = threadIdx.x % S::kLanes;
  float w[S::kVec][S::kU], b[S::kVec][S::kU];
#pragma unroll
  for (int k = 0; k < S::kVec; ++k) {
    const int c = S::kU * (l + k * S::kLanes);
    param(w[k], a.w, a.w_f32, c, a.cols, 1.0f);
    param(b[k], a.b, a.b_f32, c, a.cols, 0.0f);
  }
  const int64_t step = static_cast<int64_t>(gridDim.x) * S::kRows;
  const int mine = threadIdx.x / S::kLanes;
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * S::kRows; r0 < a.rows; r0 += step) {
    const int64_t r = r0 + mine;
    const int cols = r < a.rows ? a.cols : 0;
    float x[S::kVec][S::kU];
#pragma unroll
    for (int k = 0; k < S::kVec; ++k) {
      const int c = S::kU * (l + k * S::kLanes);
      get<kX32>(x[k], a.x, r * a.ldx + c, cols - c);
    }
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
      put<kY32>(a.y, r * a.cols + c, y, cols - c);
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

// kParams: dw and db are wanted.
template <class S, bool kX32, bool kY32, bool kLayer, bool kParams>
__global__ __launch_bounds__(S::kThreads) void norm_backward_kernel(Backward a) {
  __shared__ float room[16];
  RowSum<S::kLanes> row_sum{room};
  const int l = threadIdx.x % S::kLanes;
  float w[S::kVec][S::kU];
  float dw[kParams ? S::kVec : 1][S::kU] = {}, db[kParams && kLayer ? S::kVec : 1][S::kU] = {};
#pragma unroll
  for (int k = 0; k < S::kVec; ++k) param(w[k], a.w, a.w_f32, S::kU * (l + k * S::kLanes), a.cols, 1.0f);
  const int64_t step = static_cast<int64_t>(gridDim.x) * S::kRows;
  const int mine = threadIdx.x / S::kLanes;
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * S::kRows; r0 < a.rows; r0 += step) {
    const int64_t r = r0 + mine;
    const int cols = r < a.rows ? a.cols : 0;
    float x[S::kVec][S::kU], dy[S::kVec][S::kU];
#pragma unroll
    for (int k = 0; k < S::kVec; ++k) {
      const int c = S::kU * (l + k * S::kLanes);
      get<kX32>(x[k], a.x, r * a.ldx + c, cols - c);
      get<kY32>(dy[k], a.dy, r * a.lddy + c, cols - c);
    }
    const float rstd = cols ? a.rstd[r] : 0.0f, mean = kLayer && cols ? a.mean[r] : 0.0f;
    float sum = 0.0f, along = 0.0f;
#pragma unroll
    for (int k = 0; k < S::kVec; ++k)
#pragma unroll
      for (int i = 0; i < S::kU; ++i) {
        const float xhat = (x[k][i] - mean) * rstd, d = dy[k][i], g = d * w[k][i];
        if constexpr (kParams) {
          dw[k][i] = fmaf(d, xhat, dw[k][i]);
          if constexpr (kLayer) db[k][i] += d;
        }
        sum += g;
        along = fmaf(g, xhat, along);
        x[k][i] = xhat;
        dy[k][i] = g;
      }
    along = row_sum(along) * a.inv_cols;
    sum = kLayer ? row_sum(sum) * a.inv_cols : 0.0f;
    if (a.dx) {
#pragma unroll
      for (int k = 0; k < S::kVec; ++k) {
        const int c = S::kU * (l + k * S::kLanes);
        float dx[S::kU];
#pragma unroll
        for (int i = 0; i < S::kU; ++i) dx[i] = (dy[k][i] - fmaf(x[k][i], along, sum)) * rstd;
        put<kX32>(a.dx, r * a.cols + c, dx, cols - c);
      }
    }
  }
  if constexpr (kParams) {
    // over the workgroup's rows in order, one unit at a time: LDS holds that unit of every row
    __shared__ float part[S::kRows > 1 ? S::kRows : 1][S::kRows > 1 ? S::kLanes * S::kU : 1];
#pragma unroll
    for (int k = 0; k < S::kVec; ++k) {
      const int c = S::kU * (l + k * S::kLanes);
#pragma unroll
      for (int which = 0; which < (kLayer ? 2 : 1); ++which) {
        float* out = which ? a.db : a.dw;
        float* sums = which ? db[kLayer ? k : 0] : dw[k];
        if (!out) continue;
        out += static_cast<int64_t>(blockIdx.x) * a.cols;
        if constexpr (S::kRows == 1) {
#pragma unroll
          for (int i = 0; i < S::kU; ++i)
            if (c + i < a.cols) out[c + i] = sums[i];
        } else {
          __syncthreads();
#pragma unroll
          for (int i = 0; i < S::kU; ++i) part[mine][S::kU * l + i] = sums[i];
          __syncthreads();
          for (int i = threadIdx.x; i < S::kLanes * S::kU; i += S::kThreads) {
            float s = part[0][i];
            for (int j = 1; j < S::kRows; ++j) s += part[j][i];
            const int at = S::kU * k * S::kLanes + i;
            if (at < a.cols) out[at] = s;
          }
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
  if (c < a.cols)
    for (int i = first; i < last; ++i) s += p[static_cast<int64_t>(i) * a.cols + c];
  part[wave][l] = s;
  __syncthreads();
  if (wave || c >= a.cols) return;
  for (int i = 1; i < 16; ++i) s += part[i][l];
  if (a.f32[blockIdx.y]) static_cast<float*>(out)[c] = s;
  else static_cast<uint16_t*>(out)[c] = static_cast<uint16_t>(pack_bf16(s, s));
}

// ---------------------------------------------------------------- which shape, how many workgroups

constexpr int kMaxCols = 16384;

// f(Shape) for rows of `cols` columns: the fewest lanes and units that hold them, a row in one wave up to 6 units a lane.
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
    default: break;
  }
  if (units <= 512) return f(Shape<256, 2, kU>{});
  if (units <= 768) return f(Shape<256, 3, kU>{});
  if (units <= 1024) return f(Shape<256, 4, kU>{});
  if (units <= 1536) return f(Shape<512, 3, kU>{});
  if (units <= 2048) return f(Shape<512, 4, kU>{});
  if constexpr (kU == 4) {
    if (units <= 3072) return f(Shape<512, 6, kU>{});
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

int grid_of(int64_t rows, int per, int threads, int waves_a_cu) {
  const int64_t want = (rows + per - 1) / per, most = static_cast<int64_t>(kCus) * waves_a_cu * kWave / threads;
  return static_cast<int>(std::min(want, std::max<int64_t>(most, kCus)));
}
#ifndef FW
#define FW 16
#define BW 8
#endif
constexpr int kForwardWaves = FW, kBackwardWaves = BW;

int backward_grid(int64_t rows, int cols, bool wide) {
  int grid = 0;
  auto count = [&](auto s) {
    grid = grid_of(rows, decltype(s)::kRows, decltype(s)::kThreads, kBackwardWaves);
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
      const dim3 grid(grid_of(rows, S::kRows, S::kThreads, kForwardWaves)), block(S::kThreads);
      if (layer) hipLaunchKernelGGL((norm_forward_kernel<S, kX, kY, true>), grid, block, 0, s, a);
      else hipLaunchKernelGGL((norm_forward_kernel<S, kX, kY, false>), grid, block, 0, s, a);
      return TM_OK;
    });
  });
  return rc ? rc : launched(who);
}

size_t tm_norm_workspace_bytes(int64_t rows, int64_t cols, int x_f32, int y_f32, int layer) {
  if (rows < 1 || cols < 1 || cols > kMaxCols) return 0;
  return static_cast<size_t>(backward_grid(rows, static_cast<int>(cols), x_f32 || y_f32)) * cols * sizeof(float) * (layer ? 2 : 1);
}

int tm_norm_backward(void* d_dx, void* d_dw, void* d_db, int b_f32, const void* d_dy, int y_f32, int64_t lddy, const void* d_x,
                     int x_f32, int64_t ldx, const float* d_rstd, const float* d_mean, const void* d_w, int w_f32, int dw_f32,
                     int layer, int64_t rows, int64_t cols, void* d_ws, size_t ws_bytes, void* stream) {
  const char* who = "tm_norm_backward";
  if (int rc = check_sizes(who, rows, cols)) return rc;
  if (rows == 0) return fail(TM_EINVAL, "%s: no rows", who);
  if (!d_dy || !d_x || !d_rstd || (layer && !d_mean)) return fail(TM_EINVAL, "%s: null input", who);
  if (!layer && d_db) return fail(TM_EINVAL, "%s: an RMS norm has no bias", who);
  if ((ldx < cols || lddy < cols) && rows > 1)
    return fail(TM_EINVAL, "%s: rows %lld and %lld elements apart", who, (long long)ldx, (long long)lddy);
  if (odd(d_dx, x_f32) || odd(d_dw, dw_f32) || odd(d_db, b_f32) || odd(d_dy, y_f32) || odd(d_x, x_f32) || odd(d_w, w_f32) ||
      odd(d_rstd, true) || odd(d_mean, true))
    return fail(TM_EINVAL, "%s: a pointer that is not aligned to its elements", who);
  const bool params = d_dw || d_db;
  const size_t need = params ? tm_norm_workspace_bytes(rows, cols, x_f32, y_f32, layer) : 0;
  if (ws_bytes < need || (need && (!d_ws || odd(d_ws, true))))
    return fail(TM_EINVAL, "%s: workspace of %zu bytes, %zu needed, aligned to 4", who, d_ws ? ws_bytes : size_t(0), need);
  const int grid = backward_grid(rows, static_cast<int>(cols), x_f32 || y_f32);
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
      const dim3 blocks(grid), block(S::kThreads);
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
