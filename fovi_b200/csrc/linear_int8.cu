// Product of 8-bit tokens with 8-bit weights:
//   y[m, n] = scale[m] weight_scale[n] sum over k of q[m, k] w[n, k] + bias[n]
// The sums are exact, in 32-bit integers; what follows is float32, rounded once to y's type.
#include "product.cuh"
#include "product_simt.cuh"

namespace {

template <typename T> struct Scaled {
  T* y; int64_t pitch; const float *scale, *wscale, *bias;
  __device__ __forceinline__ void operator()(int64_t m, int n, int v, int) const {
    y[m * pitch + n] = from_float<T>(fmaf((float)v * __ldg(scale + m), __ldg(wscale + n), bias ? __ldg(bias + n) : 0.f));
  }
};

}  // namespace

extern "C" int fovi_linear_int8(const int8_t* q, int64_t tokens, int K, int64_t q_stride, const float* scale, const int8_t* weight, int N, int64_t weight_stride,
                                const float* weight_scale, const float* bias, void* y, int y_dtype, void* stream) {
  // (-128)^2 K has to stay below 2^31
  if (tokens < 0 || tokens > (1 << 30) || K < 1 || K >= 131072 || N < 1 || q_stride < 0 || weight_stride < 0 || !fovi::valid_dtype(y_dtype)) return FOVI_ERR_INVALID_ARGUMENT;
  if (tokens == 0) return FOVI_OK;
  if (!q || !scale || !weight || !weight_scale || !y) return FOVI_ERR_INVALID_ARGUMENT;
  auto st = reinterpret_cast<cudaStream_t>(stream);
  SimtArgs p{};
  p.m = tokens; p.n = N; p.k[0] = K; p.segments = 1;
  p.a[0] = fovi::Operand{q, q_stride, 1};
  p.b[0] = fovi::Operand{weight, weight_stride, 1};
  if (y_dtype == FOVI_BF16) return product_simt<int8_t, false>(p, Scaled<__nv_bfloat16>{static_cast<__nv_bfloat16*>(y), N, scale, weight_scale, bias}, st);
  return product_simt<int8_t, false>(p, Scaled<float>{static_cast<float*>(y), N, scale, weight_scale, bias}, st);
}
