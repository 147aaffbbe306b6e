// Matrix products of few tokens: what bounds them are the weights' bytes.
#pragma once
#include "product.cuh"

namespace fovi {

constexpr int FEW_TOKENS = 32;      // up to here these kernels take a product

// Rows as in TcMatrix: `pitch` values apart, on 16-byte boundaries.
struct FewRows { const void* p; int64_t pitch; };

// h = act(x Wg^T + bg) (x Wu^T + bu), bf16.
int few_gated(const FewRows& x, const FewRows& wg, const FewRows& wu, int m, int n, int k, const void* bg, const void* bu, int act, const FewRows& h, cudaStream_t st);
// y = x W^T + bias, bf16.  after_own: the launch before it in the stream is few_gated's, with the same weights in the same call.
int few_linear(const FewRows& x, const FewRows& w, int m, int n, int k, const void* bias, void* y, bool after_own, cudaStream_t st);
// y = scale wscale (q W^T) + bias, y bf16 or float32.
int few_int8(const FewRows& q, const FewRows& w, int m, int n, int k, const float* scale, const float* wscale, const float* bias, void* y, int y_dtype, cudaStream_t st);

}  // namespace fovi
