// Layer norm over the last axis of [rows, C], and its gradients:
//   y  = (x - mean) * rstd * w + b          mean, var = mean((x - mean)^2) of the row, rstd = 1 / sqrt(var + eps)
//   dx = rstd * (g - mean(g) - xh * mean(g * xh))          g = dy * w, xh = (x - mean) * rstd
//   dw = sum over rows of dy * xh,   db = sum over rows of dy
// Sums and statistics are float32; results are rounded once, to their tensor's type.  The variance is taken about the row's own mean (two passes over
// values that are already on the chip), so a large common offset does not cost digits.
#include <cuda_bf16.h>

#include "common.cuh"

namespace {

constexpr int GEN_THREADS = 256;
constexpr int STRIP_COLS = 128;      // columns of a CTA of the weight-gradient pass

__device__ __forceinline__ float block_sum(float v, float* red) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.f;
  for (int i = 0; i < GEN_THREADS / 32; ++i) t += red[i];
  return t;
}

// One CTA per row, any C.
template <typename TX, typename TY>
__global__ void __launch_bounds__(GEN_THREADS) layer_norm_kernel(const TX* x, int64_t rows, int C, int64_t stride, const float* w, const float* b, float eps, TY* y,
                                                                 float2* stats) {
  __shared__ float red[GEN_THREADS / 32];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const TX* xr = x + r * stride;
    float s = 0.f;
    for (int c = threadIdx.x; c < C; c += GEN_THREADS) s += ld_as_float(xr + c);
    const float mean = block_sum(s, red) / C;
    s = 0.f;
    for (int c = threadIdx.x; c < C; c += GEN_THREADS) { const float d = ld_as_float(xr + c) - mean; s += d * d; }
    const float rstd = 1.f / sqrtf(block_sum(s, red) / C + eps);
    if (stats && threadIdx.x == 0) stats[r] = make_float2(mean, rstd);
    for (int c = threadIdx.x; c < C; c += GEN_THREADS)
      y[r * C + c] = from_float<TY>((ld_as_float(xr + c) - mean) * rstd * (w ? __ldg(w + c) : 1.f) + (b ? __ldg(b + c) : 0.f));
  }
}

template <typename TX, typename TY>
__global__ void __launch_bounds__(GEN_THREADS) layer_norm_dx_kernel(const TX* x, int64_t rows, int C, int64_t stride, const TY* dy, int64_t dy_stride, const float* w,
                                                                    const float2* stats, TX* dx) {
  __shared__ float red[GEN_THREADS / 32];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const float2 st = __ldg(stats + r);
    float sg = 0.f, sgx = 0.f;
    for (int c = threadIdx.x; c < C; c += GEN_THREADS) {
      const float g = ld_as_float(dy + r * dy_stride + c) * (w ? __ldg(w + c) : 1.f);
      sg += g;
      sgx += g * ((ld_as_float(x + r * stride + c) - st.x) * st.y);
    }
    sg = block_sum(sg, red) / C;
    sgx = block_sum(sgx, red) / C;
    for (int c = threadIdx.x; c < C; c += GEN_THREADS) {
      const float g = ld_as_float(dy + r * dy_stride + c) * (w ? __ldg(w + c) : 1.f), xh = (ld_as_float(x + r * stride + c) - st.x) * st.y;
      dx[r * C + c] = from_float<TX>(st.y * (g - sg - xh * sgx));
    }
  }
}

// A thread per column and strip of rows: the strip's part of both sums, [strip][2][C].
template <typename TX, typename TY>
__global__ void __launch_bounds__(STRIP_COLS) layer_norm_dw_kernel(const TX* x, int64_t rows, int C, int64_t stride, const TY* dy, int64_t dy_stride, const float2* stats,
                                                                   float* part, int strips) {
  const int c = blockIdx.x * STRIP_COLS + threadIdx.x;
  if (c >= C) return;
  float sw = 0.f, sb = 0.f;
  for (int64_t r = blockIdx.y; r < rows; r += strips) {
    const float2 st = __ldg(stats + r);
    const float g = ld_as_float(dy + r * dy_stride + c);
    sw += g * ((ld_as_float(x + r * stride + c) - st.x) * st.y);
    sb += g;
  }
  part[((size_t)blockIdx.y * 2) * C + c] = sw;
  part[((size_t)blockIdx.y * 2 + 1) * C + c] = sb;
}

// The parts of every column added in the order of the strips: the same bits every time.
__global__ void __launch_bounds__(256) layer_norm_join_kernel(const float* part, int strips, int C, float* dw, float* db) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= C) return;
  float sw = 0.f, sb = 0.f;
  for (int s = 0; s < strips; ++s) {
    sw += __ldg(part + ((size_t)s * 2) * C + c);
    sb += __ldg(part + ((size_t)s * 2 + 1) * C + c);
  }
  if (dw) dw[c] = sw;
  if (db) db[c] = sb;
}

int strips_of(int64_t rows) { return (int)(rows < 512 ? (rows + 15) / 16 : 64); }

template <typename TX, typename TY>
int forward(const void* x, int64_t rows, int C, int64_t stride, const float* w, const float* b, float eps, void* y, float* stats, cudaStream_t st) {
  const int grid = (int)(rows < 148 * 8 ? rows : 148 * 8);
  layer_norm_kernel<TX, TY><<<grid, GEN_THREADS, 0, st>>>((const TX*)x, rows, C, stride, w, b, eps, (TY*)y, (float2*)stats);
  return fovi::after_launch("layer_norm_kernel");
}

template <typename TX, typename TY>
int backward(const void* x, int64_t rows, int C, int64_t stride, const void* dy, int64_t dy_stride, const float* w, const float* stats, void* dx, float* dw, float* db,
             float* work, cudaStream_t st) {
  if (dx) {
    const int grid = (int)(rows < 148 * 8 ? rows : 148 * 8);
    layer_norm_dx_kernel<TX, TY><<<grid, GEN_THREADS, 0, st>>>((const TX*)x, rows, C, stride, (const TY*)dy, dy_stride, w, (const float2*)stats, (TX*)dx);
    const int rc = fovi::after_launch("layer_norm_dx_kernel");
    if (rc) return rc;
  }
  if (dw || db) {
    const int strips = strips_of(rows);
    const dim3 grid((C + STRIP_COLS - 1) / STRIP_COLS, strips);
    layer_norm_dw_kernel<TX, TY><<<grid, STRIP_COLS, 0, st>>>((const TX*)x, rows, C, stride, (const TY*)dy, dy_stride, (const float2*)stats, work, strips);
    int rc = fovi::after_launch("layer_norm_dw_kernel");
    if (rc) return rc;
    layer_norm_join_kernel<<<(C + 255) / 256, 256, 0, st>>>(work, strips, C, dw, db);
    return fovi::after_launch("layer_norm_join_kernel");
  }
  return FOVI_OK;
}

}  // namespace

extern "C" int64_t fovi_layer_norm_workspace_bytes(int64_t rows, int C) {
  if (rows < 0 || C < 1) return -1;
  return (int64_t)strips_of(rows) * 2 * C * 4;
}

extern "C" int fovi_layer_norm_forward(const void* x, int x_dtype, int64_t rows, int C, int64_t x_stride, const float* weight, const float* bias, float eps, void* y,
                                       int y_dtype, float* stats, void* stream) {
  if (rows < 0 || C < 1 || x_stride < 0 || !(eps >= 0.f) || !fovi::valid_dtype(x_dtype) || !fovi::valid_dtype(y_dtype)) return FOVI_ERR_INVALID_ARGUMENT;
  if (rows == 0) return FOVI_OK;
  if (!x || !y) return FOVI_ERR_INVALID_ARGUMENT;
  auto st = reinterpret_cast<cudaStream_t>(stream);
  const bool xb = x_dtype == FOVI_BF16, yb = y_dtype == FOVI_BF16;
  if (xb) return yb ? forward<__nv_bfloat16, __nv_bfloat16>(x, rows, C, x_stride, weight, bias, eps, y, stats, st)
                    : forward<__nv_bfloat16, float>(x, rows, C, x_stride, weight, bias, eps, y, stats, st);
  return yb ? forward<float, __nv_bfloat16>(x, rows, C, x_stride, weight, bias, eps, y, stats, st)
            : forward<float, float>(x, rows, C, x_stride, weight, bias, eps, y, stats, st);
}

extern "C" int fovi_layer_norm_backward(const void* x, int x_dtype, int64_t rows, int C, int64_t x_stride, const void* dy, int y_dtype, int64_t dy_stride,
                                        const float* weight, const float* stats, void* dx, float* dweight, float* dbias, void* work, int64_t work_bytes, void* stream) {
  if (rows < 0 || C < 1 || x_stride < 0 || dy_stride < 0 || !fovi::valid_dtype(x_dtype) || !fovi::valid_dtype(y_dtype)) return FOVI_ERR_INVALID_ARGUMENT;
  auto st = reinterpret_cast<cudaStream_t>(stream);
  if (rows == 0) {
    if (dweight) FOVI_CUDA(cudaMemsetAsync(dweight, 0, (size_t)C * 4, st));
    if (dbias) FOVI_CUDA(cudaMemsetAsync(dbias, 0, (size_t)C * 4, st));
    return FOVI_OK;
  }
  if (!x || !dy || !stats) return FOVI_ERR_INVALID_ARGUMENT;
  if ((dweight || dbias) && (!work || work_bytes < fovi_layer_norm_workspace_bytes(rows, C))) return FOVI_ERR_INVALID_ARGUMENT;
  const bool xb = x_dtype == FOVI_BF16, yb = y_dtype == FOVI_BF16;
  float* wk = static_cast<float*>(work);
  if (xb) return yb ? backward<__nv_bfloat16, __nv_bfloat16>(x, rows, C, x_stride, dy, dy_stride, weight, stats, dx, dweight, dbias, wk, st)
                    : backward<__nv_bfloat16, float>(x, rows, C, x_stride, dy, dy_stride, weight, stats, dx, dweight, dbias, wk, st);
  return yb ? backward<float, __nv_bfloat16>(x, rows, C, x_stride, dy, dy_stride, weight, stats, dx, dweight, dbias, wk, st)
            : backward<float, float>(x, rows, C, x_stride, dy, dy_stride, weight, stats, dx, dweight, dbias, wk, st);
}
