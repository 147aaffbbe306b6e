// Matrix products on the CUDA cores: float32 arithmetic (whole numbers: 32-bit integers), any sizes and strides.
//   D[m, n] = sum over the segments s and over k of A_s[m, k] B_s[n, k]          (TWO: a second sum with B2 in B's place)
// What becomes of a sum is the epilogue's matter: a functor of (m, n, sums).
#pragma once
#include "product.cuh"

namespace {

constexpr int SP_T = 64, SP_K = 16, SP_THREADS = 256;

template <typename T> struct SumOf { using type = float; };
template <> struct SumOf<int8_t> { using type = int; };

template <typename T> __device__ __forceinline__ typename SumOf<T>::type element(const T* p) { return ld_as_float(p); }
template <> __device__ __forceinline__ int element<int8_t>(const int8_t* p) { return *p; }

struct SimtArgs {
  fovi::Operand a[2], b[2], b2;
  int64_t m; int n, k[2], segments;
};

template <typename T, typename S>
__device__ __forceinline__ void stage(S (*to)[SP_T + 4], const fovi::Operand& o, int64_t first, int64_t rows, int k0, int K) {
  const bool along_k = o.step == 1;
  for (int e = threadIdx.x; e < SP_T * SP_K; e += SP_THREADS) {
    const int i = along_k ? e / SP_K : e % SP_T, k = along_k ? e % SP_K : e / SP_T;
    to[k][i] = first + i < rows && k0 + k < K ? element<T>(static_cast<const T*>(o.p) + (first + i) * o.row + (k0 + k) * o.step) : S(0);
  }
}

template <typename T, bool TWO, typename Epilogue>
__global__ void __launch_bounds__(SP_THREADS) product_simt_kernel(const SimtArgs p, const Epilogue out) {
  using S = typename SumOf<T>::type;
  __shared__ S sa[SP_K][SP_T + 4], sb[SP_K][SP_T + 4], sc[TWO ? SP_K : 1][SP_T + 4];
  const int64_t m0 = (int64_t)blockIdx.y * SP_T;
  const int n0 = blockIdx.x * SP_T, ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  S d[4][4] = {}, d2[TWO ? 4 : 1][4] = {};
  for (int s = 0; s < p.segments; ++s)
    for (int k0 = 0; k0 < p.k[s]; k0 += SP_K) {
      __syncthreads();
      stage<T>(sa, p.a[s], m0, p.m, k0, p.k[s]);
      stage<T>(sb, p.b[s], n0, p.n, k0, p.k[s]);
      if (TWO) stage<T>(sc, p.b2, n0, p.n, k0, p.k[s]);
      __syncthreads();
#pragma unroll
      for (int k = 0; k < SP_K; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            d[i][j] += sa[k][4 * ty + i] * sb[k][4 * tx + j];
            if (TWO) d2[TWO ? i : 0][j] += sa[k][4 * ty + i] * sc[TWO ? k : 0][4 * tx + j];
          }
    }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (m0 + 4 * ty + i < p.m && n0 + 4 * tx + j < p.n) out(m0 + 4 * ty + i, n0 + 4 * tx + j, d[i][j], d2[TWO ? i : 0][j]);
}

template <typename T, bool TWO, typename Epilogue> int product_simt(const SimtArgs& p, const Epilogue& out, cudaStream_t st) {
  const int64_t rows = (p.m + SP_T - 1) / SP_T;
  if (rows > 65535) return FOVI_ERR_UNSUPPORTED;
  product_simt_kernel<T, TWO, Epilogue><<<dim3((p.n + SP_T - 1) / SP_T, (unsigned)rows), SP_THREADS, 0, st>>>(p, out);
  return fovi::after_launch("product_simt_kernel");
}

}  // namespace
