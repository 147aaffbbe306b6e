// Rotary positions with several axes.  x [B, L, H, D]; pair p of a head belongs to one axis a(p) and turns by the angle  t = position[b, l, a(p)] * frequency[p]:
//   (u, v) -> (u cos t - v sin t, v cos t + u sin t)
// `pairing` says which channels a pair is: (p, p + P) of the first 2P ("halves") or (2p, 2p + 1) ("pairs"); channels from 2P on, and the first `prefix` tokens
// (class and register tokens, which have no place), pass as they are.  The gradient is the same map with -t: a rotation's transpose.
// A token's angles are the same for all its heads.  The angle is the exact product, in two float32 parts: cos and sin are taken at the rounded product (whose
// error grows with it: 4e-6 at t = 64) and turned by its rounding error e: cos(t + e) = cos t - e sin t, sin(t + e) = sin t + e cos t, up to e^2.
#include <algorithm>
#include <limits.h>

#include <cuda_bf16.h>

#include "common.cuh"

namespace {

constexpr int MAX_AXES = 4;

struct RotArgs {
  int64_t tokens;                        // B * L
  int L, H, D, P, prefix, axes, ends[MAX_AXES], interleaved, inverse;
  int64_t sb, sl, sh, pos_batch;         // element strides of x; of a sample's positions (0: shared)
  const float *pos, *freq;
};

// place: the token's positions
__device__ __forceinline__ void turn_of(const RotArgs& a, const float* place, int p, float& c, float& s) {
  int ax = 0;
#pragma unroll
  for (int i = 0; i < MAX_AXES - 1; ++i) ax += i < a.axes - 1 && p >= a.ends[i];
  const float q = __ldg(place + ax), f = __ldg(a.freq + p);
  const float t = __fmul_rn(q, f), e = __fmaf_rn(q, f, -t);
  float s0, c0;
  sincosf(t, &s0, &c0);
  c = fmaf(-s0, e, c0);
  s = fmaf(c0, e, s0);
  if (a.inverse) s = -s;
}

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// Any strides and alignment.  One thread per (token, pair) and per channel that passes, all heads.
template <typename T>
__global__ void __launch_bounds__(256) rotary_kernel(const T* x, T* y, const RotArgs a) {
  const int per = a.D - a.P;             // P pairs, then D - 2P channels
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t token = i / per;
  if (token >= a.tokens) return;
  const int p = (int)(i - token * per), l = (int)(token % a.L);
  const int64_t b = token / a.L;
  const T* xt = x + b * a.sb + l * a.sl;
  T* yt = y + token * a.H * a.D;
  if (p >= a.P) {
    const int c = p + a.P;
    for (int h = 0; h < a.H; ++h) yt[h * a.D + c] = xt[h * a.sh + c];
    return;
  }
  const int c0 = a.interleaved ? 2 * p : p, c1 = a.interleaved ? 2 * p + 1 : p + a.P;
  if (l < a.prefix) {
    for (int h = 0; h < a.H; ++h) { yt[h * a.D + c0] = xt[h * a.sh + c0]; yt[h * a.D + c1] = xt[h * a.sh + c1]; }
    return;
  }
  float c, s;
  turn_of(a, a.pos + b * a.pos_batch + (int64_t)(l - a.prefix) * a.axes, p, c, s);
  for (int h = 0; h < a.H; ++h) {
    const float u = ld_as_float(xt + h * a.sh + c0), v = ld_as_float(xt + h * a.sh + c1);
    yt[h * a.D + c0] = from_float<T>(u * c - v * s);
    yt[h * a.D + c1] = from_float<T>(v * c + u * s);
  }
}

// Rows on 16-byte boundaries, whole pieces of V channels (16 bytes).  A block takes `tokens` tokens: their cosines and sines once, into shared memory, then all heads
// piece by piece, "halves" with the two pieces that turn together in one thread.  A thread's first PIECES pieces are on their way while the angles are worked out.
// What bounds it is a block's chain (places, barrier, loads, angles, barrier, stores), which it goes through once and which only the SM's other blocks cover, next to its instructions: issue slots
// 68 % and shared memory 65 % taken, no one kind of stall above a quarter of a warp's time (first size below).  With launches (us): 256 x 257 x 6 x 64 bf16, two axes: 25 (4.0 TB/s; a thread per pair over all heads: 50);
// 7 x 1029 x 20 x 64 float32, three axes: 18 to 19 (3.8 to 4.2 TB/s; 19 as well); 64 x 500 x 12 x 128 bf16: 40 (4.9 TB/s; 72).
struct Tile { int tokens, per, row; uint32_t by_per, by_row, by_pairs; };      // pieces of a head and of a token; 2^32 / d rounded up, for divisions of small numbers

__device__ __forceinline__ int over(int i, uint32_t by) { return (int)__umulhi((uint32_t)i, by); }

template <typename T, bool INTERLEAVED>
__global__ void __launch_bounds__(256) rotary_tile_kernel(const T* __restrict__ x, T* __restrict__ y, const RotArgs a, const Tile q) {
  constexpr int V = 16 / sizeof(T), PIECES = 2;
  extern __shared__ float2 cs[];           // [tokens][P], then where each token lies and whether it turns
  int64_t* at = reinterpret_cast<int64_t*>(cs + q.tokens * a.P);
  const int64_t t0 = (int64_t)blockIdx.x * q.tokens;
  const int n = (int)min((int64_t)q.tokens, a.tokens - t0);
  const int turning = INTERLEAVED ? 2 * a.P / V : a.P / V;
  if (threadIdx.x < n) {
    const int64_t token = t0 + threadIdx.x, b = token / a.L;
    const int l = (int)(token - b * a.L);
    at[2 * threadIdx.x] = b * a.sb + l * a.sl;
    at[2 * threadIdx.x + 1] = l < a.prefix ? -1 : b * a.pos_batch + (int64_t)(l - a.prefix) * a.axes;
  }
  __syncthreads();
  uint4 u[PIECES], v[PIECES];
  auto fetch = [&](int i, uint4& u, uint4& v) {
    const int t = over(i, q.by_row), e = i - t * q.row, h = over(e, q.by_per), k = e - h * q.per;
    const T* xt = x + at[2 * t] + h * a.sh;
    const int c0 = k < turning ? k * V : 2 * a.P + (k - turning) * V;
    u = __ldg(reinterpret_cast<const uint4*>(xt + c0));
    if (!INTERLEAVED && k < turning) v = __ldg(reinterpret_cast<const uint4*>(xt + c0 + a.P));
  };
#pragma unroll
  for (int r = 0; r < PIECES; ++r)
    if ((int)threadIdx.x + 256 * r < n * q.row) fetch(threadIdx.x + 256 * r, u[r], v[r]);
  for (int i = threadIdx.x; i < n * a.P; i += 256) {
    const int t = over(i, q.by_pairs), p = i - t * a.P;
    const int64_t place = at[2 * t + 1];
    if (place >= 0) turn_of(a, a.pos + place, p, cs[i].x, cs[i].y);
  }
  __syncthreads();
  auto finish = [&](int i, uint4 u, uint4 v) {
    const int t = over(i, q.by_row), e = i - t * q.row, h = over(e, q.by_per), k = e - h * q.per;
    T* yt = y + ((t0 + t) * a.H + h) * a.D;
    const int c0 = k < turning ? k * V : 2 * a.P + (k - turning) * V;
    if (k < turning && at[2 * t + 1] >= 0) {
      const float2* f = cs + t * a.P + (INTERLEAVED ? k * V / 2 : k * V);
      T *us = reinterpret_cast<T*>(&u), *vs = reinterpret_cast<T*>(&v);
#pragma unroll
      for (int j = 0; j < (INTERLEAVED ? V / 2 : V); ++j) {
        T &p = INTERLEAVED ? us[2 * j] : us[j], &w = INTERLEAVED ? us[2 * j + 1] : vs[j];
        const float pf = as_float(p), wf = as_float(w);
        const float2 z = f[j];
        p = from_float<T>(pf * z.x - wf * z.y);
        w = from_float<T>(wf * z.x + pf * z.y);
      }
    }
    *reinterpret_cast<uint4*>(yt + c0) = u;
    if (!INTERLEAVED && k < turning) *reinterpret_cast<uint4*>(yt + c0 + a.P) = v;
  };
#pragma unroll
  for (int r = 0; r < PIECES; ++r)
    if ((int)threadIdx.x + 256 * r < n * q.row) finish(threadIdx.x + 256 * r, u[r], v[r]);
  for (int i = threadIdx.x + 256 * PIECES; i < n * q.row; i += 256) {      // tokens of many heads
    fetch(i, u[0], v[0]);
    finish(i, u[0], v[0]);
  }
}

template <typename T>
int run(const void* x, void* y, const RotArgs& a, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const bool whole = (a.interleaved ? 2 * a.P : a.P) % V == 0 && a.D % V == 0 && 2 * a.P % V == 0 && a.sb % V == 0 && a.sl % V == 0 && a.sh % V == 0 &&
                     !((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & 15u);
  if (whole) {
    // two pieces a thread, while there are blocks enough for every SM (four each); 16 KB of cosines and sines at most
    Tile q;
    q.per = (a.interleaved ? 2 * a.P / V : a.P / V) + (a.D - 2 * a.P) / V;
    q.row = a.H * q.per;
    int64_t tokens = std::max<int64_t>(1, 512 / std::max(q.row, 1));
    tokens = std::max<int64_t>(1, std::min(tokens, a.tokens / (4 * fovi::sm_count())));
    if (a.P > 0) tokens = std::min<int64_t>(tokens, std::max(1, 2048 / a.P));
    tokens = std::min<int64_t>(tokens, 256);
    auto by = [](int d) { return d > 1 ? (uint32_t)((0xffffffffull + d) / d) : 0u; };
    q.tokens = (int)tokens; q.by_per = by(q.per); q.by_row = by(q.row); q.by_pairs = by(a.P);
    const int64_t blocks = (a.tokens + tokens - 1) / tokens;
    const size_t smem = (size_t)tokens * (a.P * sizeof(float2) + 2 * sizeof(int64_t));
    // (products of a number and its divisor stay below 2^32: the divisions are exact; a divisor of one has no such factor)
    if (blocks <= INT_MAX && smem <= 49152 && q.per > 1 && q.row > 1 && a.P > 1 && (int64_t)tokens * q.row * q.row < (1ll << 32)) {
      if (a.interleaved) rotary_tile_kernel<T, true><<<(int)blocks, 256, smem, st>>>((const T*)x, (T*)y, a, q);
      else rotary_tile_kernel<T, false><<<(int)blocks, 256, smem, st>>>((const T*)x, (T*)y, a, q);
      return fovi::after_launch("rotary_tile_kernel");
    }
  }
  const int64_t blocks = (a.tokens * (a.D - a.P) + 255) / 256;
  if (blocks > INT_MAX) return FOVI_ERR_UNSUPPORTED;
  rotary_kernel<T><<<(int)blocks, 256, 0, st>>>((const T*)x, (T*)y, a);
  return fovi::after_launch("rotary_kernel");
}

}  // namespace

extern "C" int fovi_rotary(const void* x, int dtype, int B, int L, int H, int D, const int64_t* x_strides, const float* positions, int64_t pos_batch_stride, int axes,
                           const int32_t* pairs_per_axis, const float* frequencies, int prefix, int interleaved, int inverse, void* y, void* stream) {
  if (B < 0 || L < 0 || H < 1 || D < 1 || !x_strides || axes < 1 || axes > MAX_AXES || !pairs_per_axis || prefix < 0 || prefix > L || pos_batch_stride < 0 ||
      !fovi::valid_dtype(dtype))
    return FOVI_ERR_INVALID_ARGUMENT;
  RotArgs a;
  int64_t P = 0;
  for (int i = 0; i < MAX_AXES; ++i) {
    if (i < axes && pairs_per_axis[i] < 0) return FOVI_ERR_INVALID_ARGUMENT;
    P += i < axes ? pairs_per_axis[i] : 0;
    a.ends[i] = (int)P;
    if (2 * P > D) return FOVI_ERR_INVALID_ARGUMENT;
  }
  if ((int64_t)B * L == 0) return FOVI_OK;
  if (!x || !y || (P > 0 && L > prefix && (!positions || !frequencies))) return FOVI_ERR_INVALID_ARGUMENT;
  a.tokens = (int64_t)B * L; a.L = L; a.H = H; a.D = D; a.P = (int)P; a.prefix = prefix; a.axes = axes; a.interleaved = interleaved; a.inverse = inverse;
  a.sb = x_strides[0]; a.sl = x_strides[1]; a.sh = x_strides[2]; a.pos_batch = pos_batch_stride; a.pos = positions; a.freq = frequencies;
  auto st = reinterpret_cast<cudaStream_t>(stream);
  return dtype == FOVI_BF16 ? run<__nv_bfloat16>(x, y, a, st) : run<float>(x, y, a, st);
}
