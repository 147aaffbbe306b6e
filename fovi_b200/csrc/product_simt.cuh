// Matrix products in float32 on the CUDA cores, any sizes and strides:
//   D[m, n] = sum over the segments s and over k of A_s[m, k] B_s[n, k]          (TWO: a second sum with B2 in B's place)
// What becomes of a sum is the epilogue's matter: a functor of (task, m, n, sums of four neighbouring columns, how many of them there are).
// Tiles of 64 x 64, 128 threads, 8 x 4 sums a thread, two multiply-adds an instruction (rows in pairs; a column's value is doubled in registers: 16 such instructions, 4 moves and 3
// shared-memory reads a step of k).  The next 16 of k are on their way to registers while these are worked on.  Small tiles, since what this path is for, parity runs, is small: a few
// hundred tiles fill the SMs, and k is divided among blocks where there are fewer (SPLIT; the parts are joined in their order).
#pragma once
#include <algorithm>

#include "pairs.cuh"
#include "product.cuh"

namespace {

constexpr int SP_T = 64, SP_K = 16, SP_THREADS = 128, SP_TASKS = 3, SP_PITCH = SP_T + 4;

struct SimtTask { fovi::Operand a[2], b[2], b2; int64_t m; int n, k[2]; int first, cols; };      // first: of its tiles, cols: tiles side by side
struct SimtArgs { SimtTask t[SP_TASKS]; int tasks, segments, splits, tiles; };

// Four values of an operand: along k (its k is contiguous) or along its rows.  vec: they can be had in one load.
struct Place { const float* p; int64_t row, step; bool along_k, vec; };
__device__ __forceinline__ Place place_of(const fovi::Operand& o) {
  Place q{static_cast<const float*>(o.p), o.row, o.step, o.step == 1, false};
  q.vec = (reinterpret_cast<uintptr_t>(o.p) & 15) == 0 && (q.along_k ? o.row : o.step) % 4 == 0;
  return q;
}
// Piece e (0 .. 255) of the 64 x 16 tile at (first, k0): 4 of k of a row, or 4 rows of a k.
__device__ __forceinline__ float4 fetch(const Place& o, int e, int64_t first, int64_t rows, int k0, int K) {
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  if (o.along_k) {
    const int64_t i = first + (e >> 2);
    const int k = k0 + 4 * (e & 3);
    if (i < rows && k < K) {
      const float* p = o.p + i * o.row + k;
      if (o.vec && k + 4 <= K) return __ldg(reinterpret_cast<const float4*>(p));
#pragma unroll
      for (int j = 0; j < 4; ++j) if (k + j < K) v[j] = __ldg(p + j);
    }
  } else {
    const int64_t i = first + 4 * (e & 15);
    const int k = k0 + (e >> 4);
    if (i < rows && k < K) {
      const float* p = o.p + i + k * o.step;
      if (o.vec && i + 4 <= rows) return __ldg(reinterpret_cast<const float4*>(p));
#pragma unroll
      for (int j = 0; j < 4; ++j) if (i + j < rows) v[j] = __ldg(p + j);
    }
  }
  return make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void put(float (*to)[SP_PITCH], const Place& o, int e, const float4& v) {
  if (o.along_k) {
    const int i = e >> 2, k = 4 * (e & 3);
    to[k][i] = v.x; to[k + 1][i] = v.y; to[k + 2][i] = v.z; to[k + 3][i] = v.w;
  } else {
    *reinterpret_cast<float4*>(&to[e >> 4][4 * (e & 15)]) = v;
  }
}

template <bool TWO, typename Epilogue>
__global__ void __launch_bounds__(SP_THREADS) product_simt_kernel(const __grid_constant__ SimtArgs p, const __grid_constant__ Epilogue out) {
  __shared__ __align__(16) float sa[2][SP_K][SP_PITCH], sb[2][SP_K][SP_PITCH], sc[TWO ? 2 : 1][TWO ? SP_K : 1][SP_PITCH];
  const int split = blockIdx.x / p.tiles, tile = blockIdx.x % p.tiles;
  const int task = p.tasks > 1 ? (tile >= p.t[2].first ? 2 : tile >= p.t[1].first ? 1 : 0) : 0;
  const SimtTask& t = p.t[task];
  const int64_t m0 = (int64_t)((tile - t.first) / t.cols) * SP_T;
  const int n0 = (tile - t.first) % t.cols * SP_T, ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  const int steps0 = (t.k[0] + SP_K - 1) / SP_K, steps = steps0 + (p.segments > 1 ? (t.k[1] + SP_K - 1) / SP_K : 0);
  const int from = (int)((int64_t)steps * split / p.splits), to = (int)((int64_t)steps * (split + 1) / p.splits);
  float2 d[4][4], d2[TWO ? 4 : 1][4];                    // of rows 8 ty + 2 i and the next, column 4 tx + j
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) { d[i][j] = both(0.f); d2[TWO ? i : 0][j] = both(0.f); }
  float4 ra[2], rb[2], rc[TWO ? 2 : 1];
  Place a, b, c;
  auto fetch_step = [&](int s) {
    const int seg = s >= steps0 ? 1 : 0, k0 = (s - (seg ? steps0 : 0)) * SP_K, K = t.k[seg];
    a = place_of(t.a[seg]);
    b = place_of(t.b[seg]);
    if (TWO) c = place_of(t.b2);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int e = threadIdx.x + u * SP_THREADS;
      ra[u] = fetch(a, e, m0, t.m, k0, K);
      rb[u] = fetch(b, e, n0, t.n, k0, K);
      if (TWO) rc[TWO ? u : 0] = fetch(c, e, n0, t.n, k0, K);
    }
  };
  auto stage = [&](int buf) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int e = threadIdx.x + u * SP_THREADS;
      put(sa[buf], a, e, ra[u]);
      put(sb[buf], b, e, rb[u]);
      if (TWO) put(sc[TWO ? buf : 0], c, e, rc[TWO ? u : 0]);
    }
  };
  if (from < to) { fetch_step(from); stage(from & 1); }
  __syncthreads();
  for (int s = from; s < to; ++s) {
    const int buf = s & 1;
    if (s + 1 < to) fetch_step(s + 1);
#pragma unroll
    for (int k = 0; k < SP_K; ++k) {
      const float4 a0 = *reinterpret_cast<const float4*>(&sa[buf][k][8 * ty]), a1 = *reinterpret_cast<const float4*>(&sa[buf][k][8 * ty + 4]);
      const float2 av[4] = {make_float2(a0.x, a0.y), make_float2(a0.z, a0.w), make_float2(a1.x, a1.y), make_float2(a1.z, a1.w)};
      const float4 b0 = *reinterpret_cast<const float4*>(&sb[buf][k][4 * tx]);
      const float bv[4] = {b0.x, b0.y, b0.z, b0.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i][j] = fma2(av[i], both(bv[j]), d[i][j]);
      if (TWO) {
        const float4 c0 = *reinterpret_cast<const float4*>(&sc[TWO ? buf : 0][TWO ? k : 0][4 * tx]);
        const float cv[4] = {c0.x, c0.y, c0.z, c0.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) d2[TWO ? i : 0][j] = fma2(av[i], both(cv[j]), d2[TWO ? i : 0][j]);
      }
    }
    if (s + 1 < to) stage(buf ^ 1);
    __syncthreads();
  }
  const int n = n0 + 4 * tx, left = min(4, t.n - n);
  if (left <= 0) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t m = m0 + 8 * ty + i;
    if (m >= t.m) continue;
    float v[4], u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) { v[j] = i & 1 ? d[i / 2][j].y : d[i / 2][j].x; u[j] = TWO ? (i & 1 ? d2[TWO ? i / 2 : 0][j].y : d2[TWO ? i / 2 : 0][j].x) : 0.f; }
    out(task, split, m, n, v, u, left);
  }
}

// Up to four neighbouring values, in one store where they lie for it.
__device__ __forceinline__ void store4(float* p, const float (&v)[4], int left, int64_t pitch) {
  if (left == 4 && pitch % 4 == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < left) p[j] = v[j];
  }
}

// Results with a bias, or parts of k for the join: part[task][split][m][n].
struct Store {
  float* y[SP_TASKS]; int64_t pitch[SP_TASKS], m[SP_TASKS], part[SP_TASKS]; const float* bias; float* work; int splits;
  __device__ __forceinline__ void operator()(int task, int split, int64_t r, int n, float (&v)[4], float (&)[4], int left) const {
    if (splits > 1) {
      store4(work + part[task] + ((int64_t)split * m[task] + r) * pitch[task] + n, v, left, pitch[task]);
      return;
    }
    if (bias) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < left) v[j] += __ldg(bias + n + j);
    }
    store4(y[task] + r * pitch[task] + n, v, left, pitch[task]);
  }
};
__global__ void __launch_bounds__(256) product_simt_join_kernel(const __grid_constant__ Store a) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, values = a.m[blockIdx.y] * a.pitch[blockIdx.y];
  if (i >= values) return;
  const float* from = a.work + a.part[blockIdx.y] + i;
  float s = 0.f;
  for (int p = 0; p < a.splits; ++p) s += __ldg(from + p * values);
  a.y[blockIdx.y][i] = s + (a.bias ? __ldg(a.bias + i % a.pitch[blockIdx.y]) : 0.f);
}

// Tiles of the tasks, and how many parts k is cut into: what fills the SMs four blocks deep, of 64 of k and more.  (From every task's size, whether or not its result is wanted.)
inline int simt_splits(const SimtTask* t, int n, int segments) {
  int64_t tiles = 0, k = 0;
  for (int i = 0; i < n; ++i) tiles += (t[i].m + SP_T - 1) / SP_T * ((t[i].n + SP_T - 1) / SP_T);
  for (int s = 0; s < segments; ++s) k += t[0].k[s];
  return (int)std::max<int64_t>(1, std::min<int64_t>({4ll * fovi::sm_count() / std::max<int64_t>(1, tiles), k / 64, 16}));
}

template <bool TWO, typename Epilogue> int product_simt(SimtArgs& p, const Epilogue& out, cudaStream_t st) {
  int64_t at = 0;
  for (int i = 0; i < p.tasks; ++i) {
    p.t[i].first = (int)at;
    p.t[i].cols = (p.t[i].n + SP_T - 1) / SP_T;
    at += (p.t[i].m + SP_T - 1) / SP_T * p.t[i].cols;
  }
  if (at * p.splits >= (1ll << 31)) return FOVI_ERR_UNSUPPORTED;
  for (int i = p.tasks; i < SP_TASKS; ++i) p.t[i].first = (int)at;
  p.tiles = (int)at;
  product_simt_kernel<TWO, Epilogue><<<(unsigned)(at * p.splits), SP_THREADS, 0, st>>>(p, out);
  return fovi::after_launch("product_simt_kernel");
}

// Bytes of the parts of products that simt_store cuts.
inline int64_t simt_store_bytes(const SimtTask* t, int n, int segments) {
  const int splits = simt_splits(t, n, segments);
  int64_t bytes = 0;
  for (int i = 0; splits > 1 && i < n; ++i) bytes += (int64_t)splits * t[i].m * t[i].n * 4;
  return bytes;
}

// y[i] = task i's product + bias; a task with y null is left out.
inline int simt_store(const SimtTask* t, float* const* y, int n, int segments, const float* bias, float* work, cudaStream_t st) {
  SimtArgs p{};
  Store out{};
  p.segments = segments;
  out.splits = p.splits = simt_splits(t, n, segments);
  out.bias = bias; out.work = work;
  int64_t at = 0;
  for (int i = 0; i < n; ++i) {
    if (!y[i]) continue;
    const int q = p.tasks++;
    p.t[q] = t[i];
    out.y[q] = y[i]; out.pitch[q] = t[i].n; out.m[q] = t[i].m; out.part[q] = at;
    at += (int64_t)out.splits * t[i].m * t[i].n;
  }
  if (!p.tasks) return FOVI_OK;
  const int rc = product_simt<false>(p, out, st);
  if (rc || out.splits == 1) return rc;
  int64_t most = 0;
  for (int q = 0; q < p.tasks; ++q) most = std::max(most, out.m[q] * out.pitch[q]);
  product_simt_join_kernel<<<dim3((unsigned)((most + 255) / 256), p.tasks), 256, 0, st>>>(out);
  return fovi::after_launch("product_simt_join_kernel");
}

}  // namespace
