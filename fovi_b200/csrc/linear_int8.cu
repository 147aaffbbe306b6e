// Product of 8-bit tokens with 8-bit weights:
//   y[m, n] = scale[m] weight_scale[n] sum over k of q[m, k] w[n, k] + bias[n]
// The sums are exact, in 32-bit integers; what follows is float32, rounded once to y's type.
// Bound by the tensor cores' integer rate and their operands' way through L2 for many tokens (16448 x 1280 -> 5120: 97 us, 2.2 P a second), by the weights' bytes for few (one token
// 1280 -> 5120: 3.0 to 4.5 us for 6.6 MB).
#include "product_few.cuh"
#include "product_tc.cuh"

namespace {

int linear_int8(const int8_t* q, int64_t tokens, int K, int64_t q_stride, const float* scale, const int8_t* weight, int N, int64_t weight_stride, const float* weight_scale,
                const float* bias, void* y, int y_dtype, bool selftest, void* stream) {
  // (-128)^2 K has to stay below 2^31; rows and columns are counted in 32 bits, a tile beyond the last ones
  if (tokens < 0 || tokens > (1 << 30) || K < 1 || K >= 131072 || N < 1 || N > (1 << 30) || q_stride < 0 || weight_stride < 0 || !fovi::valid_dtype(y_dtype)) return FOVI_ERR_INVALID_ARGUMENT;
  if (tokens == 0) return FOVI_OK;
  if (!q || !scale || !weight || !weight_scale || !y) return FOVI_ERR_INVALID_ARGUMENT;
  if (!fovi::tc_takes(q, q_stride, 1) || !fovi::tc_takes(weight, weight_stride, 1) || reinterpret_cast<uintptr_t>(y) % 16) return FOVI_ERR_ALIGNMENT;
  if (fovi::few_eight(tokens, K, N) && !selftest)
    return fovi::few_int8({q, q_stride}, {weight, weight_stride}, (int)tokens, N, K, scale, weight_scale, bias, y, y_dtype, reinterpret_cast<cudaStream_t>(stream));
  return fovi::tc_int8({q, tokens, K, q_stride}, {weight, N, K, weight_stride}, scale, weight_scale, bias, y, y_dtype, selftest, reinterpret_cast<cudaStream_t>(stream));
}

}  // namespace

extern "C" int fovi_linear_int8(const int8_t* q, int64_t tokens, int K, int64_t q_stride, const float* scale, const int8_t* weight, int N, int64_t weight_stride,
                                const float* weight_scale, const float* bias, void* y, int y_dtype, void* stream) {
  return linear_int8(q, tokens, K, q_stride, scale, weight, N, weight_stride, weight_scale, bias, y, y_dtype, false, stream);
}

extern "C" int fovi_linear_int8_selftest_wait_timeout(const int8_t* q, int64_t tokens, int K, int64_t q_stride, const float* scale, const int8_t* weight, int N,
                                                      int64_t weight_stride, const float* weight_scale, const float* bias, void* y, int y_dtype, void* stream) {
  return linear_int8(q, tokens, K, q_stride, scale, weight, N, weight_stride, weight_scale, bias, y, y_dtype, true, stream);
}
