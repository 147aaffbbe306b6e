// Matrix products of a token block on the tensor cores: what their entry points hand over.
#pragma once
#include "product.cuh"

namespace fovi {

// A matrix as it lies in memory: `rows` rows of `cols` values (bf16 or 8-bit integers), `pitch` values apart, on 16-byte boundaries.
struct TcMatrix { const void* p; int64_t rows, cols, pitch; };
inline bool tc_takes(const void* p, int64_t pitch, int size) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && pitch * size % 16 == 0 && pitch > 0; }

// One product of a launch: y [m, n] = A B^T, A [m, k] and B [n, k] as memory holds them, or (.._mn) their transposes.
struct TcTask { TcMatrix a, b; int m, n; void* y; };

// How a product is cut: column tiles of `ct`, K in `splits` parts.
struct TcShape { int ct, splits; };

// h = act(x Wg^T + bg) (x Wu^T + bu), and g and u where `to` has places for them.
int tc_gated(const TcMatrix& x, const TcMatrix& wg, const TcMatrix& wu, const void* bg, const void* bu, int act, const Hidden& to, cudaStream_t st);
// dg, du from dh = dy Wd and the saved g, u; with `sums` also the column sums of each 32 rows of dg and du, [ceil(rows / 32) to whole tiles][2][pitch].
int tc_hidden_grad(const TcMatrix& dy, const TcMatrix& wd, const Hidden& from, int act, void* dg, void* du, float* sums, cudaStream_t st);
int64_t tc_sum_rows(int64_t tokens);
// y = A B^T + bias, bf16; k runs over a and b, then over a2 and b2 where there are any (two segments of k each).  b_mn: B lies as [k, n].
int64_t tc_linear_bytes(int64_t m, int n, int64_t k, int segments);
int tc_linear(const TcMatrix& a, const TcMatrix& b, const TcMatrix* a2, const TcMatrix* b2, bool b_mn, int m, int n, const void* bias, void* y, void* work, cudaStream_t st);
// Up to three products y = A^T B over the rows of A and B: weight gradients over `rows` tokens.  A task with y null is left out.
int64_t tc_weight_grads_bytes(const TcTask* tasks, int n, int64_t rows);
int tc_weight_grads(const TcTask* tasks, int n, int64_t rows, void* work, cudaStream_t st);
// y[m, n] = scale[m] wscale[n] sum over k of q[m, k] w[n, k] + bias[n], y bf16 or float32.
int tc_int8(const TcMatrix& q, const TcMatrix& w, const float* scale, const float* wscale, const float* bias, void* y, int y_dtype, bool selftest, cudaStream_t st);

}  // namespace fovi
