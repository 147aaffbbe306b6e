// Cross attention of queries q [B, Lq, H, D] to an encoder's states k, v [B, Lk, Hkv, D], and its gradients, in float32 arithmetic on the CUDA cores:
// float32 inputs, and every shape, stride and alignment that the tensor-core kernels do not take.
//   s = scale * q k^T (masked keys: -inf),  p = softmax(s),  o = p v;  a row without a key gives 0
//   delta = rowsum(dy * o),  ds = p * (dy v^T - delta),  dq = scale * ds k,  dk = scale * ds^T q,  dv = p^T dy, the last two summed over the heads that
//   share a state head
// What bounds it are the shared-memory reads that feed the multiply-adds, eight of 16 bytes for 64 of them (forward: shared memory 73 % taken, multiply-add units 47 %, issue slots 67 %): 512 queries over 1024 keys, 8 x 20 heads of 64 channels: forward 722 us (30 TFLOP/s), dq
// 1099 (29), dk and dv 1412 (30).  Two blocks an SM up to 64 channels, for a few spilled registers: with one block of 150 registers the forward pass took 936 us.
// Tiles of 64 x 64 scores, 16 x 16 threads with 4 x 4 each, operands in shared memory as float32.  The forward pass goes over the keys once with the running
// maximum and sum of every row; the backward pass recomputes p from the row's logarithm of the sum.  dq goes by query tiles and dk, dv by key tiles,
// each by one CTA in a fixed order: no atomics, the same bits every time.  Masked keys are read as zeros, whatever they hold.
#include <cuda_bf16.h>

#include "attention_tc.cuh"

using fovi::AttnArgs;
using fovi::key_end;

namespace {

constexpr int T = 64;                    // queries and keys of a tile
constexpr int THREADS = 256;
constexpr int PP = T + 4;                // pitch of a tile of scores
constexpr float INF = __builtin_huge_valf();

// Keys of split `split`: the splits share out the sample's keys in whole tiles.
struct Range { int first, end; };
__device__ __forceinline__ Range keys_of(const AttnArgs& a, int end, int split, int tile) {
  const int share = ((end + tile - 1) / tile + a.splits - 1) / a.splits * tile;
  const int64_t first = (int64_t)split * share;
  return {(int)min(first, (int64_t)end), (int)min(first + share, (int64_t)end)};
}

template <int DP> constexpr int PITCH = DP + 4;        // rows 4 floats apart modulo 32 banks: eight threads' float4 reads of one column do not collide

__device__ __forceinline__ bool key_ok(const AttnArgs& a, int b, int key, int end) {
  return key < end && (!a.mask || __ldg(a.mask + (int64_t)b * a.Lk + key));
}

// A thread's part of a tile: rows [r0, r0 + 64) of one head as float32, zeros behind `n` and D.  It is fetched while the tile before it is worked on.  With `vec` the rows are whole pieces of
// 16 bytes on 16-byte boundaries.
template <typename E, int DP>
struct Part {
  static constexpr int V = 16 / sizeof(E), N = T * DP / (V * THREADS), ROW = DP / V;      // pieces of V channels
  float x[N][V];
  __device__ __forceinline__ void fetch(const E* src, int64_t sl, int r0, int n, int D, bool vec) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int i = threadIdx.x + k * THREADS, r = i / ROW, c = i % ROW * V;
      const E* p = src + (int64_t)(r0 + r) * sl + c;
#pragma unroll
      for (int e = 0; e < V; ++e) x[k][e] = 0.f;
      if (r0 + r >= n) continue;
      if (vec) {
        if (c >= D) continue;
        const uint4 w = __ldg(reinterpret_cast<const uint4*>(p));
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < V; ++e) x[k][e] = V == 4 ? __uint_as_float(u[e % 4]) : __uint_as_float(e & 1 ? u[e / 2 % 4] & 0xffff0000u : u[e / 2 % 4] << 16);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (c + e < D) x[k][e] = ld_as_float(p + e);
      }
    }
  }
  __device__ __forceinline__ void store(float* dst, const unsigned char* ok = nullptr) const {      // zeros in the rows where `ok` says no
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int i = threadIdx.x + k * THREADS, r = i / ROW, c = i % ROW * V;
      const bool in = !ok || ok[r];
#pragma unroll
      for (int e = 0; e < V; e += 4)
        *reinterpret_cast<float4*>(dst + r * PITCH<DP> + c + e) = in ? make_float4(x[k][e], x[k][e + 1], x[k][e + 2], x[k][e + 3]) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }
};

// Rounds of 16 rows that `n` rows take, four at most.
__device__ __forceinline__ int rounds(int n) { return min(4, (n + 15) / 16); }

// acc[i][j] = <A row ty + 16 i, B row tx + 16 j>, of NI and NJ rounds of rows; zeros beyond
template <int DP, int NI, int NJ>
__device__ __forceinline__ void dot_rounds(const float* A, const float* B, float (&acc)[4][4]) {
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
#pragma unroll 4
  for (int d = 0; d < DP; d += 4) {
    float4 x[NI], y[NJ];
#pragma unroll
    for (int i = 0; i < NI; ++i) x[i] = *reinterpret_cast<const float4*>(A + (ty + 16 * i) * PITCH<DP> + d);
#pragma unroll
    for (int j = 0; j < NJ; ++j) y[j] = *reinterpret_cast<const float4*>(B + (tx + 16 * j) * PITCH<DP> + d);
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        acc[i][j] = fmaf(x[i].x, y[j].x, acc[i][j]); acc[i][j] = fmaf(x[i].y, y[j].y, acc[i][j]);
        acc[i][j] = fmaf(x[i].z, y[j].z, acc[i][j]); acc[i][j] = fmaf(x[i].w, y[j].w, acc[i][j]);
      }
  }
}

// The same of a last tile's first ni, nj rounds, each taken as one, two or four (rows behind a tile's end are zeros).  One product at a
// time reads eight times as much shared memory a product: 23 queries over 621 keys, 17 x 12 heads of 128 channels, forward, dq, dk and dv: 198, 373, 324 us, so 146, 231, 211.
template <int DP>
__device__ __forceinline__ void dot_tile(const float* A, const float* B, float (&acc)[4][4], int ni, int nj) {
  if (ni > 2) {
    if (nj > 2) dot_rounds<DP, 4, 4>(A, B, acc);
    else if (nj == 2) dot_rounds<DP, 4, 2>(A, B, acc);
    else dot_rounds<DP, 4, 1>(A, B, acc);
  } else if (ni == 2) {
    if (nj > 2) dot_rounds<DP, 2, 4>(A, B, acc);
    else dot_rounds<DP, 2, 2>(A, B, acc);
  } else {
    if (nj > 2) dot_rounds<DP, 1, 4>(A, B, acc);
    else dot_rounds<DP, 1, 2>(A, B, acc);
  }
}

// acc[i][c] += sum over r of P[ty + 16 i][r] * V[r][channel c of this thread], channels 64 jj + 4 tx .. + 3; the first ni rounds of rows, 16 nr values of r
template <int DP>
__device__ __forceinline__ void mix_tile(const float* P, const float* V, float (&acc)[4][DP / 16], int ni, int nr) {
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
#pragma unroll 2
  for (int r = 0; r < 16 * nr; r += 4) {
    float4 v[4][DP / 64];
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int jj = 0; jj < DP / 64; ++jj) v[q][jj] = *reinterpret_cast<const float4*>(V + (r + q) * PITCH<DP> + 64 * jj + 4 * tx);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i >= ni) break;
      float p[4];
      *reinterpret_cast<float4*>(p) = *reinterpret_cast<const float4*>(P + (ty + 16 * i) * PP + r);
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int jj = 0; jj < DP / 64; ++jj) {
          acc[i][4 * jj] = fmaf(p[q], v[q][jj].x, acc[i][4 * jj]); acc[i][4 * jj + 1] = fmaf(p[q], v[q][jj].y, acc[i][4 * jj + 1]);
          acc[i][4 * jj + 2] = fmaf(p[q], v[q][jj].z, acc[i][4 * jj + 2]); acc[i][4 * jj + 3] = fmaf(p[q], v[q][jj].w, acc[i][4 * jj + 3]);
        }
    }
  }
}

// The sixteen threads of a row are half a warp.
__device__ __forceinline__ float row_max(float v) {
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float row_sum(float v) {
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename E, int DP>
__device__ __forceinline__ void store_tile(E* dst, int64_t pitch, int r0, int n, int D, const float (&acc)[4][DP / 16], const float (&f)[4]) {
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + ty + 16 * i;
    if (r >= n) continue;
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
      const int d = 64 * (c >> 2) + 4 * tx + (c & 3);
      if (d < D) dst[r * pitch + d] = from_float<E>(acc[i][c] * f[i]);
    }
  }
}

// ------------------------------------------------------------------------------------------------------------ forward: a CTA per (64 queries, head, sample)
template <typename E, int DP>
__global__ void __launch_bounds__(THREADS, DP <= 64 ? 2 : 1) attn_forward_kernel(const AttnArgs a) {
  extern __shared__ float4 smem4[];
  float* Q = reinterpret_cast<float*>(smem4);
  float *K = Q + T * PITCH<DP>, *V = K + T * PITCH<DP>, *P = V + T * PITCH<DP>;
  __shared__ unsigned char ok[T];
  const int n_qt = (a.Lq + T - 1) / T, ty = threadIdx.x >> 4, tx = threadIdx.x & 15, split = blockIdx.x % a.splits, block = blockIdx.x / a.splits;
  const int qt = block % n_qt, h = block / n_qt % a.H, b = block / n_qt / a.H;
  const Range range = keys_of(a, key_end(a, b), split, T);
  const int end = range.end;
  const E* k = (const E*)a.k + b * a.k_sb + (h / a.group) * a.k_sh;
  const E* v = (const E*)a.v + b * a.v_sb + (h / a.group) * a.v_sh;
  const int ni = rounds(a.Lq - qt * T);
  Part<E, DP> nk, nv;
  nv.fetch((const E*)a.q + b * a.q_sb + h * a.q_sh, a.q_sl, qt * T, a.Lq, a.D, a.vec);
  nv.store(Q);
  nk.fetch(k, a.k_sl, range.first, end, a.D, a.vec);
  nv.fetch(v, a.v_sl, range.first, end, a.D, a.vec);
  float m[4], l[4], acc[4][DP / 16];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INF; l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) acc[i][c] = 0.f;
  }
  for (int k0 = range.first; k0 < end; k0 += T) {
    const int nj = rounds(end - k0);
    __syncthreads();
    if (threadIdx.x < T) ok[threadIdx.x] = key_ok(a, b, k0 + threadIdx.x, end);
    if (a.mask) __syncthreads();
    nk.store(K, a.mask ? ok : nullptr);
    nv.store(V, a.mask ? ok : nullptr);
    __syncthreads();
    if (k0 + T < end) {
      nk.fetch(k, a.k_sl, k0 + T, end, a.D, a.vec);
      nv.fetch(v, a.v_sl, k0 + T, end, a.D, a.vec);
    }
    float s[4][4];
    dot_tile<DP>(Q, K, s, ni, nj);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float top = -INF;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = ok[tx + 16 * j] ? s[i][j] * a.scale_log2 : -INF;
        top = fmaxf(top, s[i][j]);
      }
      const float m_new = fmaxf(m[i], row_max(top)), base = m_new == -INF ? 0.f : m_new;      // no key yet: exp2(-inf - 0) = 0
      const float f = exp2f(m[i] - base);
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p = exp2f(s[i][j] - base);
        P[(ty + 16 * i) * PP + tx + 16 * j] = p;
        sum += p;
      }
      l[i] = l[i] * f + row_sum(sum);
      m[i] = m_new;
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) acc[i][c] *= f;
    }
    __syncthreads();
    mix_tile<DP>(P, V, acc, ni, nj);
  }
  float inv[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // (no key: the sum is zero; scores that are all not a number leave no maximum either, but a sum that is none, and so are the result and its logarithm)
    const bool none = m[i] == -INF && !(l[i] != l[i]);
    inv[i] = none ? 0.f : 1.f / l[i];
    const int r = qt * T + ty + 16 * i;
    const float lse = none ? INF : m[i] + log2f(l[i]);
    if (tx == 0 && r < a.Lq) {
      if (a.splits > 1) a.part_lse[(((int64_t)split * a.B + b) * a.Lq + r) * a.H + h] = lse;
      else if (a.lse) a.lse[((int64_t)b * a.H + h) * a.Lq + r] = lse;
    }
  }
  const int64_t at = ((int64_t)b * a.Lq * a.H + h) * a.D, pitch = (int64_t)a.H * a.D;
  if (a.splits > 1) store_tile<float, DP>(a.part_o + (int64_t)split * a.B * a.Lq * pitch + at, pitch, qt * T, a.Lq, a.D, acc, inv);
  else store_tile<E, DP>((E*)a.out + at, pitch, qt * T, a.Lq, a.D, acc, inv);
}

// A block per query (few of them: a tile would stand nearly empty): DP / 4 lanes hold a key's channels, four each, and take every 8th (4th above 64 channels) key of the block's, four at a
// time so that their loads are on the way together.  Memory bounds it: keys and values are read once per query, of the same sample and head one after another.  One query over 2056 keys,
// 64 x 20 heads, float32: 202 us, 6.7 TB/s (as a tile of 64: 1056).  Eight queries over 700, 8 x 12 heads: 40 us, as much as sixteen take as a tile (39): the rule's bound.
constexpr int FEW = 8, FEW_THREADS = 128, FEW_KEYS = 4;

template <typename E>
__device__ __forceinline__ float4 load4(const E* p, int c, int D, bool vec) {
  float x[4] = {0.f, 0.f, 0.f, 0.f};
  if (vec && c < D) {
    if constexpr (sizeof(E) == 4) {
      return __ldg(reinterpret_cast<const float4*>(p + c));
    } else {
      const uint2 w = __ldg(reinterpret_cast<const uint2*>(p + c));
      return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (c + e < D) x[e] = ld_as_float(p + c + e);
  return make_float4(x[0], x[1], x[2], x[3]);
}

template <typename E, int DP>
__global__ void __launch_bounds__(FEW_THREADS) attn_few_kernel(const AttnArgs a) {
  constexpr int LANES = DP / 4, GROUPS = FEW_THREADS / LANES;
  __shared__ __align__(8) float part[GROUPS][DP + 2];
  const int split = blockIdx.x % a.splits, block = blockIdx.x / a.splits;
  const int q = block % a.Lq, h = block / a.Lq % a.H, b = block / a.Lq / a.H, group = threadIdx.x / LANES, c = threadIdx.x % LANES * 4;
  const Range range = keys_of(a, key_end(a, b), split, FEW_KEYS * GROUPS);
  const E* k = (const E*)a.k + b * a.k_sb + (h / a.group) * a.k_sh;
  const E* v = (const E*)a.v + b * a.v_sb + (h / a.group) * a.v_sh;
  const float4 x = load4((const E*)a.q + b * a.q_sb + (int64_t)q * a.q_sl + h * a.q_sh, c, a.D, a.vec);
  float m = -INF, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k0 = range.first + group; k0 - group < range.end; k0 += FEW_KEYS * GROUPS) {       // (all lanes of a warp the same number of times)
    float s[FEW_KEYS];
    float4 y[FEW_KEYS], z[FEW_KEYS];
    bool in[FEW_KEYS];
#pragma unroll
    for (int u = 0; u < FEW_KEYS; ++u) {
      const int key = k0 + u * GROUPS;
      in[u] = key_ok(a, b, key, range.end);
      y[u] = z[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (in[u]) {
        y[u] = load4(k + (int64_t)key * a.k_sl, c, a.D, a.vec);
        z[u] = load4(v + (int64_t)key * a.v_sl, c, a.D, a.vec);
      }
    }
    float top = m;
#pragma unroll
    for (int u = 0; u < FEW_KEYS; ++u) {
      s[u] = fmaf(x.w, y[u].w, fmaf(x.z, y[u].z, fmaf(x.y, y[u].y, x.x * y[u].x)));
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) s[u] += __shfl_xor_sync(0xffffffffu, s[u], o);
      s[u] = in[u] ? s[u] * a.scale_log2 : -INF;
      top = fmaxf(top, s[u]);
    }
    const float base = top == -INF ? 0.f : top, f = exp2f(m - base);
    m = top;
    l *= f;
    acc.x *= f; acc.y *= f; acc.z *= f; acc.w *= f;
#pragma unroll
    for (int u = 0; u < FEW_KEYS; ++u) {
      const float p = exp2f(s[u] - base);
      l += p;
      acc.x = fmaf(p, z[u].x, acc.x); acc.y = fmaf(p, z[u].y, acc.y); acc.z = fmaf(p, z[u].z, acc.z); acc.w = fmaf(p, z[u].w, acc.w);
    }
  }
  *reinterpret_cast<float2*>(&part[group][c]) = make_float2(acc.x, acc.y);
  *reinterpret_cast<float2*>(&part[group][c + 2]) = make_float2(acc.z, acc.w);
  if (c == 0) { part[group][DP] = m; part[group][DP + 1] = l; }
  __syncthreads();
  if (threadIdx.x >= a.D) return;
  float top = -INF, sum = 0.f, o = 0.f;
  for (int g = 0; g < GROUPS; ++g) top = fmaxf(top, part[g][DP]);
  const float base = top == -INF ? 0.f : top;
  for (int g = 0; g < GROUPS; ++g) {
    const float f = exp2f(part[g][DP] - base);
    sum = fmaf(f, part[g][DP + 1], sum);
    o = fmaf(f, part[g][threadIdx.x], o);
  }
  // (no key: the sum is zero; scores that are not a number: so is it)
  const bool none = top == -INF && !(sum != sum);
  const float res = none ? 0.f : o / sum, lse = none ? INF : base + log2f(sum);
  const int64_t row = ((int64_t)b * a.Lq + q) * a.H + h, rows = (int64_t)a.B * a.Lq * a.H;
  if (a.splits > 1) {
    a.part_o[(split * rows + row) * a.D + threadIdx.x] = res;
    if (threadIdx.x == 0) a.part_lse[split * rows + row] = lse;
  } else {
    ((E*)a.out)[row * a.D + threadIdx.x] = from_float<E>(res);
    if (a.lse && threadIdx.x == 0) a.lse[((int64_t)b * a.H + h) * a.Lq + q] = lse;
  }
}

// The parts of a row over the splits of its keys, weighted with the parts' sums, added in their order.  A thread per channel.
template <typename E>
__global__ void __launch_bounds__(256) attn_join_parts_kernel(const AttnArgs a) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, rows = (int64_t)a.B * a.Lq * a.H, row = i / a.D;
  if (row >= rows) return;
  float top = -INF, sum = 0.f, o = 0.f;                    // a part without a key has +inf in place of its logarithm
  for (int s = 0; s < a.splits; ++s) {
    const float v = __ldg(a.part_lse + s * rows + row);
    top = v == INF ? top : v != v ? v : fmaxf(top, v);
  }
  for (int s = 0; s < a.splits; ++s) {
    const float v = __ldg(a.part_lse + s * rows + row);
    if (v == INF) continue;
    const float w = exp2f(v - top);
    o = fmaf(w, __ldg(a.part_o + s * rows * a.D + i), o);
    sum += w;
  }
  const bool none = top == -INF;
  ((E*)a.out)[i] = from_float<E>(none ? 0.f : o / sum);
  if (a.lse && i - row * a.D == 0) {
    const int h = (int)(row % a.H);
    const int64_t bl = row / a.H, b = bl / a.Lq;
    a.lse[(b * a.H + h) * a.Lq + (bl - b * a.Lq)] = none ? INF : top + log2f(sum);
  }
}

// ------------------------------------------------------------------------------------------------------------ backward
// A warp per row: delta = <dy, o>.
template <typename E>
__global__ void __launch_bounds__(256) attn_delta_kernel(const AttnArgs a) {
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);        // b, l, h
  if (row >= (int64_t)a.B * a.Lq * a.H) return;
  const int h = (int)(row % a.H), lane = threadIdx.x & 31;
  const int64_t bl = row / a.H, b = bl / a.Lq, l = bl - b * a.Lq;
  const E* o = (const E*)a.o + row * a.D;
  const E* g = (const E*)a.dy + b * a.g_sb + l * a.g_sl + h * a.g_sh;
  float s = 0.f;
  for (int d = lane; d < a.D; d += 32) s = fmaf(ld_as_float(o + d), ld_as_float(g + d), s);
  for (int w = 16; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
  if (lane == 0) a.delta[(b * a.H + h) * a.Lq + l] = s;
}

// A CTA per (64 queries, head, sample): dq.
template <typename E, int DP>
__global__ void __launch_bounds__(THREADS, DP <= 64 ? 2 : 1) attn_dq_kernel(const AttnArgs a) {
  extern __shared__ float4 smem4[];
  float* Q = reinterpret_cast<float*>(smem4);
  float *G = Q + T * PITCH<DP>, *K = G + T * PITCH<DP>, *V = K + T * PITCH<DP>, *P = V + T * PITCH<DP>;
  __shared__ unsigned char ok[T];
  const int n_qt = (a.Lq + T - 1) / T, ty = threadIdx.x >> 4, tx = threadIdx.x & 15, split = blockIdx.x % a.splits, block = blockIdx.x / a.splits;
  const int qt = block % n_qt, h = block / n_qt % a.H, b = block / n_qt / a.H, keys = key_end(a, b);
  const Range range = keys_of(a, keys, split, T);
  const int end = range.end;
  const E* k = (const E*)a.k + b * a.k_sb + (h / a.group) * a.k_sh;
  const E* v = (const E*)a.v + b * a.v_sb + (h / a.group) * a.v_sh;
  const int ni = rounds(a.Lq - qt * T);
  Part<E, DP> nk, nv;
  nk.fetch((const E*)a.q + b * a.q_sb + h * a.q_sh, a.q_sl, qt * T, a.Lq, a.D, a.vec);
  nv.fetch((const E*)a.dy + b * a.g_sb + h * a.g_sh, a.g_sl, qt * T, a.Lq, a.D, a.vec);
  nk.store(Q);
  nv.store(G);
  nk.fetch(k, a.k_sl, range.first, end, a.D, a.vec);
  nv.fetch(v, a.v_sl, range.first, end, a.D, a.vec);
  float lse[4], delta[4], acc[4][DP / 16], f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = qt * T + ty + 16 * i;
    const int64_t at = ((int64_t)b * a.H + h) * a.Lq + r;
    lse[i] = r < a.Lq ? __ldg(a.lse + at) : INF;
    delta[i] = r < a.Lq ? a.delta[at] : 0.f;
    f[i] = keys == 1 ? 0.f : a.scale;       // one key: its weight is one whatever its score
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) acc[i][c] = 0.f;
  }
  for (int k0 = range.first; k0 < end; k0 += T) {
    const int nj = rounds(end - k0);
    __syncthreads();
    if (threadIdx.x < T) ok[threadIdx.x] = key_ok(a, b, k0 + threadIdx.x, end);
    if (a.mask) __syncthreads();
    nk.store(K, a.mask ? ok : nullptr);
    nv.store(V, a.mask ? ok : nullptr);
    __syncthreads();
    if (k0 + T < end) {
      nk.fetch(k, a.k_sl, k0 + T, end, a.D, a.vec);
      nv.fetch(v, a.v_sl, k0 + T, end, a.D, a.vec);
    }
    float s[4][4], dp[4][4];
    dot_tile<DP>(Q, K, s, ni, nj);
    dot_tile<DP>(G, V, dp, ni, nj);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p = ok[tx + 16 * j] ? exp2f(s[i][j] * a.scale_log2 - lse[i]) : 0.f;
        P[(ty + 16 * i) * PP + tx + 16 * j] = ok[tx + 16 * j] ? p * (dp[i][j] - delta[i]) : 0.f;
      }
    __syncthreads();
    mix_tile<DP>(P, K, acc, ni, nj);
  }
  const int64_t at = ((int64_t)b * a.Lq * a.H + h) * a.D, pitch = (int64_t)a.H * a.D;
  if (a.splits > 1) store_tile<float, DP>(a.part_o + (int64_t)split * a.B * a.Lq * pitch + at, pitch, qt * T, a.Lq, a.D, acc, f);
  else store_tile<E, DP>((E*)a.dq + at, pitch, qt * T, a.Lq, a.D, acc, f);
}

// dq's parts over the splits of the keys, added in their order.  A thread per channel.
template <typename E>
__global__ void __launch_bounds__(256) attn_sum_parts_kernel(const AttnArgs a) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, n = (int64_t)a.B * a.Lq * a.H * a.D;
  if (i >= n) return;
  float sum = 0.f;
  for (int s = 0; s < a.splits; ++s) sum += __ldg(a.part_o + s * n + i);
  ((E*)a.dq)[i] = from_float<E>(sum);
}

// A CTA per (64 keys, state head, sample): dk and dv, over all queries of all heads that read the state head.
template <typename E, int DP>
__global__ void __launch_bounds__(THREADS, DP <= 64 ? 2 : 1) attn_dkv_kernel(const AttnArgs a) {
  extern __shared__ float4 smem4[];
  float* K = reinterpret_cast<float*>(smem4);
  float *V = K + T * PITCH<DP>, *Q = V + T * PITCH<DP>, *G = Q + T * PITCH<DP>, *P = G + T * PITCH<DP>, *S = P + T * PP;
  __shared__ unsigned char ok[T];
  const int n_kt = (a.Lk + T - 1) / T, ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  const int kt = blockIdx.x % n_kt, hk = blockIdx.x / n_kt % a.Hkv, b = blockIdx.x / n_kt / a.Hkv, end = key_end(a, b);
  float dk[4][DP / 16], dv[4][DP / 16], f[4], one[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[i] = end == 1 ? 0.f : a.scale; one[i] = 1.f;
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) dk[i][c] = dv[i][c] = 0.f;
  }
  if (threadIdx.x < T) ok[threadIdx.x] = key_ok(a, b, kt * T + threadIdx.x, end);
  __syncthreads();
  const int ni = rounds(min(end, a.Lk) - kt * T);
  Part<E, DP> nq, ng;
  nq.fetch((const E*)a.k + b * a.k_sb + hk * a.k_sh, a.k_sl, kt * T, end, a.D, a.vec);
  ng.fetch((const E*)a.v + b * a.v_sb + hk * a.v_sh, a.v_sl, kt * T, end, a.D, a.vec);
  nq.store(K, ok);
  ng.store(V, ok);
  const int n_qt = (a.Lq + T - 1) / T, steps = kt * T < end ? a.group * n_qt : 0;         // a tile behind the sample's length has gradients of zero
  auto fetch = [&](int i) {
    const int h = hk * a.group + i / n_qt, q0 = i % n_qt * T;
    nq.fetch((const E*)a.q + b * a.q_sb + h * a.q_sh, a.q_sl, q0, a.Lq, a.D, a.vec);
    ng.fetch((const E*)a.dy + b * a.g_sb + h * a.g_sh, a.g_sl, q0, a.Lq, a.D, a.vec);
  };
  if (steps) fetch(0);
  for (int i0 = 0; i0 < steps; ++i0) {
      const int h = hk * a.group + i0 / n_qt, q0 = i0 % n_qt * T, nj = rounds(a.Lq - q0);
      __syncthreads();
      nq.store(Q);
      ng.store(G);
      __syncthreads();
      if (i0 + 1 < steps) fetch(i0 + 1);
      float s[4][4], dp[4][4];
      dot_tile<DP>(K, Q, s, ni, nj);
      dot_tile<DP>(V, G, dp, ni, nj);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = q0 + tx + 16 * j;
        const int64_t at = ((int64_t)b * a.H + h) * a.Lq + r;
        const float lse = r < a.Lq ? __ldg(a.lse + at) : INF, delta = r < a.Lq ? a.delta[at] : 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool in = ok[ty + 16 * i];
          const float p = in ? exp2f(s[i][j] * a.scale_log2 - lse) : 0.f;
          P[(ty + 16 * i) * PP + tx + 16 * j] = p;
          S[(ty + 16 * i) * PP + tx + 16 * j] = in ? p * (dp[i][j] - delta) : 0.f;
        }
      }
      __syncthreads();
      mix_tile<DP>(P, G, dv, ni, nj);
      mix_tile<DP>(S, Q, dk, ni, nj);
    }
  // a masked key's weights are zeros, but zero times a query that is not a number is none: its gradients are set to zero
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (!ok[ty + 16 * i]) {
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) dk[i][c] = dv[i][c] = 0.f;
    }
  const int64_t at = ((int64_t)b * a.Lk * a.Hkv + hk) * a.D, pitch = (int64_t)a.Hkv * a.D;
  if (a.dk) store_tile<E, DP>((E*)a.dk + at, pitch, kt * T, a.Lk, a.D, dk, f);
  store_tile<E, DP>((E*)a.dv + at, pitch, kt * T, a.Lk, a.D, dv, one);
}

// ------------------------------------------------------------------------------------------------------------ host
template <int DP> constexpr size_t FWD_SMEM = (3 * T * PITCH<DP> + T * PP) * sizeof(float);
template <int DP> constexpr size_t DQ_SMEM = (4 * T * PITCH<DP> + T * PP) * sizeof(float);
template <int DP> constexpr size_t DKV_SMEM = (4 * T * PITCH<DP> + 2 * T * PP) * sizeof(float);

template <typename Kernel>
int launch(Kernel kernel, int64_t blocks, size_t smem, cudaStream_t st, const AttnArgs& a, const char* name) {
  if (blocks > INT_MAX) return FOVI_ERR_UNSUPPORTED;
  if (smem) FOVI_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  kernel<<<(int)blocks, THREADS, smem, st>>>(a);
  return fovi::after_launch(name);
}

// Parts of a row's keys (forward, and dq; 8 queries over 3000, 2 x 16 heads: dq 258 us in one part, 71 so; 100 over 900, 4 x 8: 128 and 71), so that the blocks fill the SMs: the number for which the rounds of blocks are shortest, each as long as its tiles and a beginning and an end of about two;
// joining the parts is about two more.  Few queries: 16 blocks an SM, as long as a part keeps 128 keys; else two an SM (one above 64 channels).
int splits_of(int B, int Lq, int Lk, int H, int D, bool few) {
  const int64_t blocks = (int64_t)B * H * (few ? Lq : (Lq + T - 1) / T), slots = (int64_t)fovi::sm_count() * (few ? 16 : D <= 64 ? 2 : 1);
  const int tile = few ? 128 : T, tiles = (Lk + tile - 1) / tile;
  int best = 1;
  int64_t least = INT64_MAX;
  for (int s = 1; s <= 32 && s <= tiles; ++s) {
    const int64_t time = (blocks * s + slots - 1) / slots * ((tiles + s - 1) / s + 2) + (s > 1 ? 2 : 0);
    if (time < least) { least = time; best = s; }
  }
  return best;
}

// The backward workspace: delta, and behind it, on a 16-byte boundary, dq's parts.  bf16 has none: here it is what the tensor cores do not take, and their workspace need not grow for it.
int64_t delta_floats(int B, int Lq, int H) { return fovi::attention_tc_backward_bytes(B, Lq, H) / 16 * 4 + 4; }
int dq_splits(int B, int Lq, int Lk, int H, int D, bool f32) { return f32 && Lk > 0 ? splits_of(B, Lq, Lk, H, D, false) : 1; }

template <typename E, int DP>
int forward(AttnArgs a, void* work, cudaStream_t st) {
  a.splits = work ? splits_of(a.B, a.Lq, a.Lk, a.H, a.D, a.Lq <= FEW) : 1;
  a.part_o = static_cast<float*>(work);
  a.part_lse = a.part_o + (int64_t)a.splits * a.B * a.Lq * a.H * a.D;
  int rc;
  if (a.Lq <= FEW) {
    const int64_t blocks = (int64_t)a.B * a.H * a.Lq * a.splits;
    if (blocks > INT_MAX) return FOVI_ERR_UNSUPPORTED;
    attn_few_kernel<E, DP><<<(int)blocks, FEW_THREADS, 0, st>>>(a);
    rc = fovi::after_launch("attn_few_kernel");
  } else {
    rc = launch(attn_forward_kernel<E, DP>, (int64_t)((a.Lq + T - 1) / T) * a.H * a.B * a.splits, FWD_SMEM<DP>, st, a, "attn_forward_kernel");
  }
  if (rc || a.splits == 1) return rc;
  return launch(attn_join_parts_kernel<E>, ((int64_t)a.B * a.Lq * a.H * a.D + 255) / 256, 0, st, a, "attn_join_parts_kernel");
}

template <typename E, int DP>
int backward(AttnArgs a, cudaStream_t st) {
  a.splits = dq_splits(a.B, a.Lq, a.Lk, a.H, a.D, sizeof(E) == 4);
  a.part_o = a.delta + delta_floats(a.B, a.Lq, a.H);
  int rc = launch(attn_delta_kernel<E>, ((int64_t)a.B * a.Lq * a.H + 7) / 8, 0, st, a, "attn_delta_kernel");
  if (!rc && a.dq) rc = launch(attn_dq_kernel<E, DP>, (int64_t)((a.Lq + T - 1) / T) * a.H * a.B * a.splits, DQ_SMEM<DP>, st, a, "attn_dq_kernel");
  if (!rc && a.dq && a.splits > 1) rc = launch(attn_sum_parts_kernel<E>, ((int64_t)a.B * a.Lq * a.H * a.D + 255) / 256, 0, st, a, "attn_sum_parts_kernel");
  if (!rc && a.dv) rc = launch(attn_dkv_kernel<E, DP>, (int64_t)((a.Lk + T - 1) / T) * a.Hkv * a.B, DKV_SMEM<DP>, st, a, "attn_dkv_kernel");
  return rc;
}

bool shape_ok(int dtype, int B, int Lq, int Lk, int H, int Hkv, int D, const int64_t* strides, int n) {
  if (!fovi::valid_dtype(dtype) || B < 0 || Lq < 0 || Lk < 0 || H < 1 || Hkv < 1 || D < 1 || H % Hkv || !strides) return false;
  for (int i = 0; i < n; ++i)
    if (strides[i] < 0) return false;
  return true;
}

AttnArgs arguments(const void* q, const void* k, const void* v, int dtype, int B, int Lq, int Lk, int H, int Hkv, int D, const int64_t* s, const int32_t* lengths,
                   const uint8_t* mask, float scale) {
  AttnArgs a = {};
  a.q = q; a.k = k; a.v = v; a.lengths = lengths; a.mask = mask;
  a.q_sb = s[0]; a.q_sl = s[1]; a.q_sh = s[2]; a.k_sb = s[3]; a.k_sl = s[4]; a.k_sh = s[5]; a.v_sb = s[6]; a.v_sl = s[7]; a.v_sh = s[8];
  a.B = B; a.Lq = Lq; a.Lk = Lk; a.H = H; a.Hkv = Hkv; a.D = D; a.group = H / Hkv;
  const int size = (int)fovi::dtype_size(dtype);
  auto whole = [&](const void* p, const int64_t* s) {
    return !((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(s[0] * size) | (uintptr_t)(s[1] * size) | (uintptr_t)(s[2] * size)) & 15u);
  };
  a.vec = D * size % 16 == 0 && whole(q, s) && whole(k, s + 3) && whole(v, s + 6);
  a.scale = scale; a.scale_log2 = scale * 1.44269504088896340736f;
  return a;
}
void gradients(AttnArgs& a, int dtype, const void* o, const void* dy, const int64_t* s, const float* lse, void* dq, void* dk, void* dv, void* work) {
  a.o = o; a.dy = dy; a.lse = const_cast<float*>(lse); a.dq = dq; a.dk = a.Lk > 0 ? dk : nullptr; a.dv = a.Lk > 0 ? dv : nullptr; a.delta = static_cast<float*>(work);
  a.g_sb = s[9]; a.g_sl = s[10]; a.g_sh = s[11];
  const int size = (int)fovi::dtype_size(dtype);
  a.vec = a.vec && !((reinterpret_cast<uintptr_t>(dy) | (uintptr_t)(s[9] * size) | (uintptr_t)(s[10] * size) | (uintptr_t)(s[11] * size)) & 15u);
}

}  // namespace

extern "C" int64_t fovi_attention_workspace_bytes(int dtype, int B, int Lq, int Lk, int H, int Hkv, int D, int backward) {
  const int64_t none = 0;
  if (!shape_ok(dtype, B, Lq, Lk, H, Hkv, D, &none, 0)) return -1;
  if (backward) {
    const int s = D > fovi::ATT_MAX_DIM || (int64_t)B * Lq == 0 ? 1 : dq_splits(B, Lq, Lk, H, D, dtype != FOVI_BF16);
    return s == 1 ? fovi::attention_tc_backward_bytes(B, Lq, H) : (delta_floats(B, Lq, H) + (int64_t)s * B * Lq * H * D) * 4;      // (of the first, delta is a part)
  }
  if (Lk < 1 || D > fovi::ATT_MAX_DIM) return 0;
  const int s = splits_of(B, Lq, Lk, H, D, Lq <= FEW);                       // of the plain kernels, which any call may come to
  const int64_t plain = s == 1 ? 0 : (int64_t)s * B * Lq * H * (D + 1) * 4;
  return dtype == FOVI_BF16 && D % 8 == 0 ? std::max(plain, fovi::attention_tc_forward_bytes(B, Lq, Lk, H, D)) : plain;
}

extern "C" int fovi_attention_forward(const void* q, const void* k, const void* v, int dtype, int B, int Lq, int Lk, int H, int Hkv, int D, const int64_t* strides,
                                      const int32_t* key_lengths, const uint8_t* key_mask, float scale, void* o, float* lse, void* work, int64_t work_bytes,
                                      void* stream) {
  if (!shape_ok(dtype, B, Lq, Lk, H, Hkv, D, strides, 9)) return FOVI_ERR_INVALID_ARGUMENT;
  if (D > fovi::ATT_MAX_DIM) return FOVI_ERR_UNSUPPORTED;
  if ((int64_t)B * Lq == 0) return FOVI_OK;
  if (!q || !o || (Lk > 0 && (!k || !v))) return FOVI_ERR_INVALID_ARGUMENT;
  const int64_t need = fovi_attention_workspace_bytes(dtype, B, Lq, Lk, H, Hkv, D, 0);
  if (need > 0 && (!work || work_bytes < need)) return FOVI_ERR_INVALID_ARGUMENT;
  AttnArgs a = arguments(q, k, v, dtype, B, Lq, Lk, H, Hkv, D, strides, key_lengths, key_mask, scale);
  a.out = o; a.lse = lse;
  auto st = reinterpret_cast<cudaStream_t>(stream);
  if (fovi::attention_tc_takes(a, dtype, false)) return fovi::launch_attention_tc_forward(a, need > 0 ? work : nullptr, st, false);
  void* room = need > 0 ? work : nullptr;
  if (dtype == FOVI_BF16) return D <= 64 ? forward<__nv_bfloat16, 64>(a, room, st) : forward<__nv_bfloat16, 128>(a, room, st);
  return D <= 64 ? forward<float, 64>(a, room, st) : forward<float, 128>(a, room, st);
}

extern "C" int fovi_attention_backward(const void* q, const void* k, const void* v, const void* o, const void* dy, int dtype, int B, int Lq, int Lk, int H, int Hkv, int D,
                                       const int64_t* strides, const int32_t* key_lengths, const uint8_t* key_mask, float scale, const float* lse, void* dq, void* dk,
                                       void* dv, void* work, int64_t work_bytes, void* stream) {
  if (!shape_ok(dtype, B, Lq, Lk, H, Hkv, D, strides, 12) || (dk && !dv)) return FOVI_ERR_INVALID_ARGUMENT;
  if (D > fovi::ATT_MAX_DIM) return FOVI_ERR_UNSUPPORTED;
  auto st = reinterpret_cast<cudaStream_t>(stream);
  if ((int64_t)B * Lq == 0) {       // no query: no gradient reaches the states
    const size_t bytes = (size_t)B * Lk * Hkv * D * fovi::dtype_size(dtype);
    if (dk && bytes) FOVI_CUDA(cudaMemsetAsync(dk, 0, bytes, st));
    if (dv && bytes) FOVI_CUDA(cudaMemsetAsync(dv, 0, bytes, st));
    return FOVI_OK;
  }
  if (!q || !o || !dy || !lse || (Lk > 0 && (!k || !v))) return FOVI_ERR_INVALID_ARGUMENT;
  const int64_t need = fovi_attention_workspace_bytes(dtype, B, Lq, Lk, H, Hkv, D, 1);
  if (need > 0 && (!work || work_bytes < need)) return FOVI_ERR_INVALID_ARGUMENT;
  AttnArgs a = arguments(q, k, v, dtype, B, Lq, Lk, H, Hkv, D, strides, key_lengths, key_mask, scale);
  gradients(a, dtype, o, dy, strides, lse, dq, dk, dv, work);
  if (fovi::attention_tc_takes(a, dtype, true)) return fovi::launch_attention_tc_backward(a, work, st, false);
  if (dtype == FOVI_BF16) return D <= 64 ? backward<__nv_bfloat16, 64>(a, st) : backward<__nv_bfloat16, 128>(a, st);
  return D <= 64 ? backward<float, 64>(a, st) : backward<float, 128>(a, st);
}

extern "C" int fovi_attention_check(void* stream) { return fovi::attention_tc_check(reinterpret_cast<cudaStream_t>(stream)); }

extern "C" int fovi_attention_forward_selftest_wait_timeout(const void* q, const void* k, const void* v, int B, int Lq, int Lk, int H, int Hkv, int D,
                                                            const int64_t* strides, float scale, void* o, void* stream) {
  if (!shape_ok(FOVI_BF16, B, Lq, Lk, H, Hkv, D, strides, 9) || !q || !k || !v || !o || (int64_t)B * Lq * Lk == 0) return FOVI_ERR_INVALID_ARGUMENT;
  AttnArgs a = arguments(q, k, v, FOVI_BF16, B, Lq, Lk, H, Hkv, D, strides, nullptr, nullptr, scale);
  a.out = o;
  if (!fovi::attention_tc_takes(a, FOVI_BF16, false)) return FOVI_ERR_UNSUPPORTED;
  return fovi::launch_attention_tc_forward(a, nullptr, reinterpret_cast<cudaStream_t>(stream), true);
}

extern "C" int fovi_attention_backward_selftest_wait_timeout(const void* q, const void* k, const void* v, const void* o, const void* dy, int B, int Lq, int Lk, int H, int Hkv,
                                                             int D, const int64_t* strides, float scale, const float* lse, void* dq, void* dk, void* dv, void* work,
                                                             int64_t work_bytes, void* stream) {
  if (!shape_ok(FOVI_BF16, B, Lq, Lk, H, Hkv, D, strides, 12) || !q || !k || !v || !o || !dy || !lse || !dk != !dv || (int64_t)B * Lq * Lk == 0 || !work ||
      work_bytes < fovi_attention_workspace_bytes(FOVI_BF16, B, Lq, Lk, H, Hkv, D, 1))
    return FOVI_ERR_INVALID_ARGUMENT;
  AttnArgs a = arguments(q, k, v, FOVI_BF16, B, Lq, Lk, H, Hkv, D, strides, nullptr, nullptr, scale);
  gradients(a, FOVI_BF16, o, dy, strides, lse, dq, dk, dv, work);
  if (!fovi::attention_tc_takes(a, FOVI_BF16, true)) return FOVI_ERR_UNSUPPORTED;
  return fovi::launch_attention_tc_backward(a, work, reinterpret_cast<cudaStream_t>(stream), true);
}
