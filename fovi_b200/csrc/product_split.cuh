// Float32 matrix products on the tensor cores: what their entry points hand over.
#pragma once
#include "product.cuh"

namespace fovi {

// A float32 matrix in three bf16 parts, x = p0 + p1 + p2: each `rows` rows of `cols` values, `pitch` values apart (a multiple of 8), one part behind the other.
struct SplitMatrix { void* p; int64_t rows, cols, pitch; };
inline int64_t split_pitch(int64_t cols) { return (cols + 7) / 8 * 8; }

// The parts of up to five matrices, in one launch.
constexpr int SPLITS_MOST = 5;
struct SplitTask { const float* x; int64_t stride; SplitMatrix to; };
int split_matrices(const SplitTask* t, int n, cudaStream_t st);

struct SplitProduct { SplitMatrix a, b; int m, n; float* y; };       // as TcTask

// g, u (float32 [rows, pitch], both null where no gradient is wanted) and h = act(g) u in parts, from x, Wg, Wu in parts.
int split_gated(const SplitMatrix& x, const SplitMatrix& wg, const SplitMatrix& wu, const float* bg, const float* bu, int act, float* g, float* u, const SplitMatrix& h, cudaStream_t st);
// dg, du in parts from dh = dy Wd and g, u.
int split_hidden_grad(const SplitMatrix& dy, const SplitMatrix& wd, const float* g, const float* u, int act, const SplitMatrix& dg, const SplitMatrix& du, cudaStream_t st);
// y = A B^T + bias; k runs over a and b, then over a2 and b2 where there are any.  b_mn: B lies as [k, n].
int64_t split_linear_bytes(int64_t m, int n, int64_t k, int segments);
int split_linear(const SplitMatrix& a, const SplitMatrix& b, const SplitMatrix* a2, const SplitMatrix* b2, bool b_mn, int m, int n, const float* bias, float* y, void* work, cudaStream_t st);
// Up to three products y = A^T B over the rows of A and B.  A task with y null is left out.
int64_t split_weight_grads_bytes(const SplitProduct* t, int n, int64_t rows);
int split_weight_grads(const SplitProduct* t, int n, int64_t rows, void* work, cudaStream_t st);
int split_status(int** word);        // the current device's status word

}  // namespace fovi
