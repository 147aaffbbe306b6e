// Root-mean-square norm over the last axis of [rows, C], of t = x, or of t = x + residual rounded to their type (the residual stream as it is stored), and its gradients:
//   y  = t * rstd * w                       rstd = 1 / sqrt(mean(t^2) + eps)
//   dt = rstd * (g - th * mean(g * th)) + (the stream's own gradient)          g = dy * w, th = t * rstd;  dx = dresidual = dt
//   dw = sum over rows of dy * th
// or y in 8 bits: q = round(y / scale), scale = max(max |y| of the row / 127, the smallest normal number).  Sums and statistics are float32; y is not rounded before it is quantised.
#include <algorithm>

#include <cuda_bf16.h>

#include "common.cuh"
#include "pairs.cuh"

namespace {

constexpr int GEN_THREADS = 256;
constexpr int STRIP_COLS = 128;      // columns of a CTA of the weight-gradient pass
constexpr float TINY = 1.17549435e-38f;

struct RmsArgs {
  const void *x, *res; int64_t rows; int C; int64_t x_stride, r_stride;
  const float* w; float eps;
  void *total, *y; int8_t* q; int64_t q_stride; float *scale, *rstd;
};
struct RmsGradArgs {
  const void *t, *dy, *dt; int64_t rows; int C; int64_t t_stride, dy_stride, dt_stride;
  const float *w, *rstd;
  void* dx; float* part;
};

// The larger of two, not a number where one is not.
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// A row's scale from its largest magnitude: infinity and not-a-number stay that, and the row's products with them.
__device__ __forceinline__ float scale_of(float most) { return max_nan(most / 127.f, TINY); }
__device__ __forceinline__ int eight_bits(float y, float inv) { return max(-127, min(127, __float2int_rn(y * inv))); }

template <bool MAX> __device__ __forceinline__ float block_join(float v, float* red) {
  for (int o = 16; o > 0; o >>= 1) { const float u = __shfl_xor_sync(0xffffffffu, v, o); v = MAX ? max_nan(v, u) : v + u; }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.f;
  for (int i = 0; i < GEN_THREADS / 32; ++i) t = MAX ? max_nan(t, red[i]) : t + red[i];
  return t;
}

// One CTA per row, any C.  NORM false: the row as it is, in 8 bits.
template <typename T, bool NORM>
__global__ void __launch_bounds__(GEN_THREADS) rms_norm_kernel(const RmsArgs a) {
  __shared__ float red[GEN_THREADS / 32];
  const int C = a.C;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* xr = static_cast<const T*>(a.x) + r * a.x_stride;
    const T* rr = a.res ? static_cast<const T*>(a.res) + r * a.r_stride : nullptr;
    auto value = [&](int c) { return rr ? ld_as_float(xr + c) + ld_as_float(rr + c) : ld_as_float(xr + c); };
    auto stored = [&](int c) {
      const T t = from_float<T>(value(c));
      return sizeof(T) == 2 ? __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(&t)) : *reinterpret_cast<const float*>(&t);
    };
    float rstd = 1.f;
    if (NORM) {
      float s = 0.f;
      for (int c = threadIdx.x; c < C; c += GEN_THREADS) {
        const float t = stored(c);
        if (a.total) static_cast<T*>(a.total)[r * C + c] = from_float<T>(t);
        s = fmaf(t, t, s);
      }
      rstd = 1.f / sqrtf(block_join<false>(s, red) / C + a.eps);
      if (a.rstd && threadIdx.x == 0) a.rstd[r] = rstd;
    }
    auto result = [&](int c) { return NORM ? stored(c) * rstd * (a.w ? __ldg(a.w + c) : 1.f) : ld_as_float(xr + c); };
    if (a.q) {
      float m = 0.f;
      for (int c = threadIdx.x; c < C; c += GEN_THREADS) m = max_nan(m, fabsf(result(c)));
      const float scale = scale_of(block_join<true>(m, red)), inv = 1.f / scale;
      if (threadIdx.x == 0) a.scale[r] = scale;
      for (int c = threadIdx.x; c < C; c += GEN_THREADS) a.q[r * a.q_stride + c] = (int8_t)eight_bits(result(c), inv);
    } else {
      for (int c = threadIdx.x; c < C; c += GEN_THREADS) static_cast<T*>(a.y)[r * C + c] = from_float<T>(result(c));
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(GEN_THREADS) rms_norm_dx_kernel(const RmsGradArgs a) {
  __shared__ float red[GEN_THREADS / 32];
  const int C = a.C;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T *tr = static_cast<const T*>(a.t) + r * a.t_stride, *gr = static_cast<const T*>(a.dy) + r * a.dy_stride;
    const T* sr = a.dt ? static_cast<const T*>(a.dt) + r * a.dt_stride : nullptr;
    const float rstd = __ldg(a.rstd + r);
    float s = 0.f;
    for (int c = threadIdx.x; c < C; c += GEN_THREADS) s = fmaf(ld_as_float(gr + c) * (a.w ? __ldg(a.w + c) : 1.f), ld_as_float(tr + c) * rstd, s);
    s = block_join<false>(s, red) / C;
    for (int c = threadIdx.x; c < C; c += GEN_THREADS) {
      const float g = ld_as_float(gr + c) * (a.w ? __ldg(a.w + c) : 1.f);
      static_cast<T*>(a.dx)[r * C + c] = from_float<T>(fmaf(rstd, g - ld_as_float(tr + c) * rstd * s, sr ? ld_as_float(sr + c) : 0.f));
    }
  }
}

// A thread per column and strip of rows: the strip's part of dw, [strip][C].
template <typename T>
__global__ void __launch_bounds__(STRIP_COLS) rms_norm_dw_kernel(const RmsGradArgs a, int strips) {
  const int c = blockIdx.x * STRIP_COLS + threadIdx.x;
  if (c >= a.C) return;
  float s = 0.f;
  for (int64_t r = blockIdx.y; r < a.rows; r += strips)
    s = fmaf(ld_as_float(static_cast<const T*>(a.dy) + r * a.dy_stride + c), ld_as_float(static_cast<const T*>(a.t) + r * a.t_stride + c) * __ldg(a.rstd + r), s);
  a.part[(size_t)blockIdx.y * a.C + c] = s;
}

// The parts of dw added in a fixed order, the same bits every time: a block takes 32 columns, 32 warps every 32nd part.
__global__ void __launch_bounds__(1024) rms_norm_join_kernel(const float* part, int parts, int C, float* dw) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < C)
    for (int p = w; p < parts; p += 32) s += part[(size_t)p * C + c];
  red[w][lane] = s;
  __syncthreads();
  if (w || c >= C) return;
  s = 0.f;
  for (int i = 0; i < 32; ++i) s += red[i][lane];
  dw[c] = s;
}

int strips_of(int64_t rows) { return (int)(rows < 512 ? (rows + 15) / 16 : 64); }

template <typename T, bool NORM> int forward(const RmsArgs& a, cudaStream_t st) {
  const int grid = (int)std::min<int64_t>(a.rows, fovi::sm_count() * 8);
  rms_norm_kernel<T, NORM><<<grid, GEN_THREADS, 0, st>>>(a);
  return fovi::after_launch("rms_norm_kernel");
}

template <typename T> int backward(const RmsGradArgs& a, float* dw, cudaStream_t st) {
  if (a.dx) {
    const int grid = (int)std::min<int64_t>(a.rows, fovi::sm_count() * 8);
    rms_norm_dx_kernel<T><<<grid, GEN_THREADS, 0, st>>>(a);
    const int rc = fovi::after_launch("rms_norm_dx_kernel");
    if (rc) return rc;
  }
  if (!dw) return FOVI_OK;
  const int strips = strips_of(a.rows);
  rms_norm_dw_kernel<T><<<dim3((a.C + STRIP_COLS - 1) / STRIP_COLS, strips), STRIP_COLS, 0, st>>>(a, strips);
  const int rc = fovi::after_launch("rms_norm_dw_kernel");
  if (rc) return rc;
  rms_norm_join_kernel<<<(a.C + 31) / 32, 1024, 0, st>>>(a.part, strips, a.C, dw);
  return fovi::after_launch("rms_norm_join_kernel");
}

}  // namespace

extern "C" int fovi_rms_norm_forward(const void* x, int dtype, int64_t rows, int C, int64_t x_stride, const void* residual, int64_t residual_stride, const float* weight,
                                     float eps, void* total, void* y, int8_t* q, int64_t q_stride, float* scale, float* rstd, void* stream) {
  if (rows < 0 || C < 1 || x_stride < 0 || residual_stride < 0 || !(eps >= 0.f) || !fovi::valid_dtype(dtype)) return FOVI_ERR_INVALID_ARGUMENT;
  if (rows == 0) return FOVI_OK;
  if (!x || (y != nullptr) == (q != nullptr) || (q && (!scale || q_stride < C)) || (residual != nullptr) != (total != nullptr)) return FOVI_ERR_INVALID_ARGUMENT;
  const RmsArgs a{x, residual, rows, C, x_stride, residual_stride, weight, eps, total, y, q, q_stride, scale, rstd};
  auto st = reinterpret_cast<cudaStream_t>(stream);
  return dtype == FOVI_BF16 ? forward<__nv_bfloat16, true>(a, st) : forward<float, true>(a, st);
}

extern "C" int fovi_quantize_rows(const void* x, int dtype, int64_t rows, int C, int64_t x_stride, int8_t* q, int64_t q_stride, float* scale, void* stream) {
  if (rows < 0 || C < 1 || x_stride < 0 || q_stride < C || !fovi::valid_dtype(dtype)) return FOVI_ERR_INVALID_ARGUMENT;
  if (rows == 0) return FOVI_OK;
  if (!x || !q || !scale) return FOVI_ERR_INVALID_ARGUMENT;
  const RmsArgs a{x, nullptr, rows, C, x_stride, 0, nullptr, 0.f, nullptr, nullptr, q, q_stride, scale, nullptr};
  auto st = reinterpret_cast<cudaStream_t>(stream);
  return dtype == FOVI_BF16 ? forward<__nv_bfloat16, false>(a, st) : forward<float, false>(a, st);
}

extern "C" int64_t fovi_rms_norm_workspace_bytes(int64_t rows, int C) {
  if (rows < 0 || C < 1) return -1;
  return (int64_t)strips_of(rows) * C * 4;
}

extern "C" int fovi_rms_norm_backward(const void* t, int dtype, int64_t rows, int C, int64_t t_stride, const void* dy, int64_t dy_stride, const void* dt, int64_t dt_stride,
                                      const float* weight, const float* rstd, void* dx, float* dweight, void* work, int64_t work_bytes, void* stream) {
  if (rows < 0 || C < 1 || t_stride < 0 || dy_stride < 0 || dt_stride < 0 || !fovi::valid_dtype(dtype)) return FOVI_ERR_INVALID_ARGUMENT;
  auto st = reinterpret_cast<cudaStream_t>(stream);
  if (rows == 0) {
    if (dweight) FOVI_CUDA(cudaMemsetAsync(dweight, 0, (size_t)C * 4, st));
    return FOVI_OK;
  }
  if (!t || !dy || !rstd) return FOVI_ERR_INVALID_ARGUMENT;
  if (dweight && (!work || work_bytes < fovi_rms_norm_workspace_bytes(rows, C))) return FOVI_ERR_INVALID_ARGUMENT;
  const RmsGradArgs a{t, dy, dt, rows, C, t_stride, dy_stride, dt_stride, weight, rstd, dx, static_cast<float*>(work)};
  return dtype == FOVI_BF16 ? backward<__nv_bfloat16>(a, dweight, st) : backward<float>(a, dweight, st);
}
