// Root-mean-square norm over the last axis of [rows, C], of t = x, or of t = x + residual rounded to their type (the residual stream as it is stored), and its gradients:
//   y  = t * rstd * w                       rstd = 1 / sqrt(mean(t^2) + eps)
//   dt = rstd * (g - th * mean(g * th)) + (the stream's own gradient)          g = dy * w, th = t * rstd;  dx = dresidual = dt
//   dw = sum over rows of dy * th
// or y in 8 bits: scale = max(max |y| of the row / 127, the smallest normal number), q = round(y * (1 / scale)): a reciprocal a row and a product a value,
// beside a half one step from round(y / scale).  Sums and statistics are float32; y is not rounded before it is quantised.
#include <algorithm>
#include <type_traits>

#include <cuda_bf16.h>

#include "common.cuh"
#include "rows.cuh"

namespace {

constexpr int GEN_THREADS = 256;
constexpr int STRIP_COLS = 128;      // columns of a CTA of the weight-gradient pass
constexpr float TINY = 1.17549435e-38f;
constexpr int MOST_CHANNELS = 1 << 30;     // columns are counted in 32 bits, a block's width beyond the last one

struct RmsArgs {
  const void *x, *res; int64_t rows; int C; int64_t x_stride, r_stride;
  const float* w; float eps;
  void *total, *y; int8_t* q; int64_t q_stride; float *scale, *rstd;
};
struct RmsGradArgs {
  const void *t, *dy, *dt; int64_t rows; int C; int64_t t_stride, dy_stride, dt_stride;
  const float *w, *rstd;
  void* dx; float* part;
};

// The larger of two, not a number where one is not.
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// A row's scale from its largest magnitude: infinity and not-a-number stay that, and the row's products with them.
__device__ __forceinline__ float scale_of(float most) { return max_nan(most / 127.f, TINY); }
__device__ __forceinline__ int eight_bits(float y, float inv) { return max(-127, min(127, __float2int_rn(y * inv))); }

template <bool MAX> __device__ __forceinline__ float block_join(float v, float* red) {
  for (int o = 16; o > 0; o >>= 1) { const float u = __shfl_xor_sync(0xffffffffu, v, o); v = MAX ? max_nan(v, u) : v + u; }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.f;
  for (int i = 0; i < GEN_THREADS / 32; ++i) t = MAX ? max_nan(t, red[i]) : t + red[i];
  return t;
}

// One CTA per row, any C.  NORM false: the row as it is, in 8 bits.
template <typename T, bool NORM>
__global__ void __launch_bounds__(GEN_THREADS) rms_norm_kernel(const RmsArgs a) {
  __shared__ float red[GEN_THREADS / 32];
  const int C = a.C;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* xr = static_cast<const T*>(a.x) + r * a.x_stride;
    const T* rr = a.res ? static_cast<const T*>(a.res) + r * a.r_stride : nullptr;
    auto value = [&](int c) { return rr ? ld_as_float(xr + c) + ld_as_float(rr + c) : ld_as_float(xr + c); };
    auto stored = [&](int c) {
      const T t = from_float<T>(value(c));
      return sizeof(T) == 2 ? __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(&t)) : *reinterpret_cast<const float*>(&t);
    };
    float rstd = 1.f;
    if (NORM) {
      float s = 0.f;
      for (int c = threadIdx.x; c < C; c += GEN_THREADS) {
        const float t = stored(c);
        if (a.total) static_cast<T*>(a.total)[r * C + c] = from_float<T>(t);
        s = fmaf(t, t, s);
      }
      rstd = 1.f / sqrtf(block_join<false>(s, red) / C + a.eps);
      if (a.rstd && threadIdx.x == 0) a.rstd[r] = rstd;
    }
    auto result = [&](int c) { return NORM ? stored(c) * rstd * (a.w ? __ldg(a.w + c) : 1.f) : ld_as_float(xr + c); };
    if (a.q) {
      float m = 0.f;
      for (int c = threadIdx.x; c < C; c += GEN_THREADS) m = max_nan(m, fabsf(result(c)));
      const float scale = scale_of(block_join<true>(m, red)), inv = 1.f / scale;
      if (threadIdx.x == 0) a.scale[r] = scale;
      for (int c = threadIdx.x; c < C; c += GEN_THREADS) a.q[r * a.q_stride + c] = (int8_t)eight_bits(result(c), inv);
    } else {
      for (int c = threadIdx.x; c < C; c += GEN_THREADS) static_cast<T*>(a.y)[r * C + c] = from_float<T>(result(c));
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(GEN_THREADS) rms_norm_dx_kernel(const RmsGradArgs a) {
  __shared__ float red[GEN_THREADS / 32];
  const int C = a.C;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T *tr = static_cast<const T*>(a.t) + r * a.t_stride, *gr = static_cast<const T*>(a.dy) + r * a.dy_stride;
    const T* sr = a.dt ? static_cast<const T*>(a.dt) + r * a.dt_stride : nullptr;
    const float rstd = __ldg(a.rstd + r);
    float s = 0.f;
    for (int c = threadIdx.x; c < C; c += GEN_THREADS) s = fmaf(ld_as_float(gr + c) * (a.w ? __ldg(a.w + c) : 1.f), ld_as_float(tr + c) * rstd, s);
    s = block_join<false>(s, red) / C;
    for (int c = threadIdx.x; c < C; c += GEN_THREADS) {
      const float g = ld_as_float(gr + c) * (a.w ? __ldg(a.w + c) : 1.f);
      static_cast<T*>(a.dx)[r * C + c] = from_float<T>(fmaf(rstd, g - ld_as_float(tr + c) * rstd * s, sr ? ld_as_float(sr + c) : 0.f));
    }
  }
}

// A thread per column and strip of rows: the strip's part of dw, [strip][C].
template <typename T>
__global__ void __launch_bounds__(STRIP_COLS) rms_norm_dw_kernel(const RmsGradArgs a, int strips) {
  const int c = blockIdx.x * STRIP_COLS + threadIdx.x;
  if (c >= a.C) return;
  float s = 0.f;
  for (int64_t r = blockIdx.y; r < a.rows; r += strips)
    s = fmaf(ld_as_float(static_cast<const T*>(a.dy) + r * a.dy_stride + c), ld_as_float(static_cast<const T*>(a.t) + r * a.t_stride + c) * __ldg(a.rstd + r), s);
  a.part[(size_t)blockIdx.y * a.C + c] = s;
}

// The parts of dw added in a fixed order, the same bits every time: a block takes 32 columns, 32 warps every 32nd part.
__global__ void __launch_bounds__(1024) rms_norm_join_kernel(const float* part, int parts, int C, float* dw) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < C)
    for (int p = w; p < parts; p += 32) s += part[(size_t)p * C + c];
  red[w][lane] = s;
  __syncthreads();
  if (w || c >= C) return;
  s = 0.f;
  for (int i = 0; i < 32; ++i) s += red[i][lane];
  dw[c] = s;
}

// ------------------------------------------------------------------------------------------------------------ rows in registers
// A row is held in registers by a team of threads (rows.cuh), a warp or, where it is too long for one, a block; the next row's loads are issued before this row's sums.  One pass over memory
// in both directions: the residual's sum, its norm and the 8-bit form with its scale come from the same registers, and the backward kernel keeps every column's part of dw over all its rows.
// What bounds it is memory: 263168 x 384 bf16 with the residual 124 us forward (6.5 TB/s) and 129 to 151 backward (5.4 and more), 65792 x 1280 into 8 bits 101 (5.8);
// quantised without a norm 40 (6.3), from float32 81 (5.2).
template <typename T, int VEC> __device__ __forceinline__ void store_eight(int8_t* p, const float* v, float inv) {
  if constexpr (VEC == 1) {
    p[0] = (int8_t)eight_bits(v[0], inv);
  } else {
    uint32_t w[VEC / 4];
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i)
      w[i] = (uint32_t)(eight_bits(v[4 * i], inv) & 0xff) | (uint32_t)(eight_bits(v[4 * i + 1], inv) & 0xff) << 8 | (uint32_t)(eight_bits(v[4 * i + 2], inv) & 0xff) << 16 |
             (uint32_t)(eight_bits(v[4 * i + 3], inv)) << 24;
    if constexpr (VEC == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(p) = w[0];
  }
}
template <typename T> __device__ __forceinline__ float rounded(float v) { return sizeof(T) == 2 ? __bfloat162float(__float2bfloat16_rn(v)) : v; }
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

enum { PLAIN = 0, EIGHT = 1, ROWS = 2 };      // y in its type; in 8 bits; x itself in 8 bits, without a norm

template <typename T, int VEC, int CH, bool BLOCK, bool RES, int FORM>
__global__ void __launch_bounds__(BLOCK ? BLOCK_MOST<VEC> : 256) rms_norm_rows_kernel(const RmsArgs a) {
  constexpr int E = CH * VEC;
  __shared__ float part[2][32], most_of[2][32];
  const Team<VEC, BLOCK> t;
  const int C = a.C, lane = threadIdx.x & 31;
  const T *x = static_cast<const T*>(a.x), *res = static_cast<const T*>(a.res);
  float wv[E];
  Piece<T, VEC> next[CH] = {}, more[RES ? CH : 1] = {};        // pieces behind the row's end stay zeros
  int pieces = 0;
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    pieces += t.first + k * t.pitch < C;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int c = t.first + k * t.pitch + i;
      wv[k * VEC + i] = FORM != ROWS && a.w && c < C ? __ldg(a.w + c) : 1.f;
    }
  }
  auto fetch = [&](int64_t r) {
#pragma unroll
    for (int k = 0; k < CH; ++k)
      if (k < pieces) {
        next[k] = load_piece<T, VEC>(x + r * a.x_stride + t.first + k * t.pitch);
        if (RES) more[RES ? k : 0] = load_piece<T, VEC>(res + r * a.r_stride + t.first + k * t.pitch);
      }
  };
  if (t.row < a.rows) fetch(t.row);
  const float inv_n = 1.f / C;
  int flip = 0;
  for (int64_t r = t.row; r < a.rows; r += t.step, flip ^= 1) {
    float v[E];
#pragma unroll
    for (int k = 0; k < CH; ++k) widen<T, VEC>(next[k], v + k * VEC);
    if (RES) {
#pragma unroll
      for (int k = 0; k < CH; ++k) {
        float u[VEC];
        widen<T, VEC>(more[RES ? k : 0], u);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[k * VEC + i] = rounded<T>(v[k * VEC + i] + u[i]);
        if (k < pieces) store_piece<T, VEC>(static_cast<T*>(a.total) + r * C + t.first + k * t.pitch, v + k * VEC);
      }
    }
    if (r + t.step < a.rows) fetch(r + t.step);
    if (FORM != ROWS) {
      float s = 0.f, s1 = 0.f;
#pragma unroll
      for (int i = 0; i < E; i += 2) { s = fmaf(v[i], v[i], s); if (i + 1 < E) s1 = fmaf(v[i + 1], v[i + 1], s1); }
      s = warp_sum(s + s1);
      if (BLOCK) {
        if (lane == 0) part[flip][t.warp] = s;
        __syncthreads();      // (two sets of parts: a warp that is ahead writes the other one)
        s = warp_sum(lane < t.warps ? part[flip][lane] : 0.f);
      }
      const float rstd = 1.f / sqrtf(fmaf(s, inv_n, a.eps));
      if (a.rstd && (BLOCK ? threadIdx.x : lane) == 0) a.rstd[r] = rstd;
#pragma unroll
      for (int i = 0; i < E; ++i) v[i] = v[i] * rstd * wv[i];
    }
    if (FORM == PLAIN) {
#pragma unroll
      for (int k = 0; k < CH; ++k)
        if (k < pieces) store_piece<T, VEC>(static_cast<T*>(a.y) + r * C + t.first + k * t.pitch, v + k * VEC);
    } else {
      float most = 0.f;
#pragma unroll
      for (int i = 0; i < E; ++i) most = max_nan(most, fabsf(v[i]));
      most = warp_max(most);
      if (BLOCK) {
        if (lane == 0) most_of[flip][t.warp] = most;
        __syncthreads();
        most = warp_max(lane < t.warps ? most_of[flip][lane] : 0.f);
      }
      const float scale = scale_of(most), inv = 1.f / scale;
      if ((BLOCK ? threadIdx.x : lane) == 0) a.scale[r] = scale;
#pragma unroll
      for (int k = 0; k < CH; ++k)
        if (k < pieces) store_eight<T, VEC>(a.q + r * a.q_stride + t.first + k * t.pitch, v + k * VEC, inv);
    }
  }
}

template <typename T, int VEC, int CH, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? BLOCK_MOST<VEC> : 256) rms_norm_grad_rows_kernel(const RmsGradArgs a) {
  constexpr int E = CH * VEC;
  __shared__ float sums[2][32];
  extern __shared__ float4 joined4[];        // warp teams: the weights (in shared memory: registers are short), then the warps' parts
  float* joined = reinterpret_cast<float*>(joined4);
  const Team<VEC, BLOCK> t;
  const int C = a.C, lane = threadIdx.x & 31;
  const T *tv = static_cast<const T*>(a.t), *dy = static_cast<const T*>(a.dy), *dt = static_cast<const T*>(a.dt);
  float wv[BLOCK ? E : 1], aw[E];
  Piece<T, VEC> nt[CH] = {}, ng[CH] = {}, ns[CH] = {};
  int pieces = 0;
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    pieces += t.first + k * t.pitch < C;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int c = t.first + k * t.pitch + i;
      if (BLOCK) wv[BLOCK ? k * VEC + i : 0] = a.w && c < C ? __ldg(a.w + c) : 1.f;
      aw[k * VEC + i] = 0.f;
    }
  }
  if (!BLOCK) {
    for (int c = threadIdx.x; c < C; c += blockDim.x) joined[c] = a.w ? __ldg(a.w + c) : 1.f;
    __syncthreads();
  }
  float nr = 0.f;
  auto fetch = [&](int64_t r) {
    nr = __ldg(a.rstd + r);
#pragma unroll
    for (int k = 0; k < CH; ++k)
      if (k < pieces) {
        nt[k] = load_piece<T, VEC>(tv + r * a.t_stride + t.first + k * t.pitch);
        ng[k] = load_piece<T, VEC>(dy + r * a.dy_stride + t.first + k * t.pitch);
        if (dt) ns[k] = load_piece<T, VEC>(dt + r * a.dt_stride + t.first + k * t.pitch);
      }
  };
  if (t.row < a.rows) fetch(t.row);
  const float inv_n = 1.f / C;
  int flip = 0;
  for (int64_t r = t.row; r < a.rows; r += t.step, flip ^= 1) {
    const float rstd = nr;
    float th[E], g[E], s = 0.f;
    Piece<T, VEC> own[CH];
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      widen<T, VEC>(nt[k], th + k * VEC);
      widen<T, VEC>(ng[k], g + k * VEC);
      own[k] = ns[k];
    }
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      if (k < pieces) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const int e = k * VEC + i;
          th[e] *= rstd;
          aw[e] = fmaf(g[e], th[e], aw[e]);
          g[e] *= BLOCK ? wv[BLOCK ? e : 0] : joined[t.first + k * t.pitch + i];
          s = fmaf(g[e], th[e], s);
        }
      }
    }
    if (r + t.step < a.rows) fetch(r + t.step);
    s = warp_sum(s);
    if (BLOCK) {
      if (lane == 0) sums[flip][t.warp] = s;
      __syncthreads();
      s = warp_sum(lane < t.warps ? sums[flip][lane] : 0.f);
    }
    s *= inv_n;
    if (a.dx) {
#pragma unroll
      for (int k = 0; k < CH; ++k) {
        if (k < pieces) {
          float o[VEC];
          widen<T, VEC>(own[k], o);
#pragma unroll
          for (int i = 0; i < VEC; ++i) o[i] = fmaf(rstd, fmaf(-th[k * VEC + i], s, g[k * VEC + i]), o[i]);
          store_piece<T, VEC>(static_cast<T*>(a.dx) + r * C + t.first + k * t.pitch, o);
        }
      }
    }
  }
  if (!a.part) return;
  float* mine = a.part + (size_t)blockIdx.x * C;
  if (BLOCK) {
#pragma unroll
    for (int k = 0; k < CH; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int c = t.first + k * t.pitch + i;
        if (c < C) mine[c] = aw[k * VEC + i];
      }
    return;
  }
  __syncthreads();                         // the weights have been read
  for (int u = 0; u < t.warps; ++u) {      // the warps' parts one after another: a fixed order
    if (t.warp == u) {
#pragma unroll
      for (int k = 0; k < CH; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const int c = t.first + k * t.pitch + i;
          if (c < C) joined[c] = (u ? joined[c] : 0.f) + aw[k * VEC + i];
        }
    }
    __syncthreads();
  }
  for (int c = threadIdx.x; c < C; c += blockDim.x) mine[c] = joined[c];
}

// Values a thread of a warp's row.  In 8 bits a block would pass two barriers a row, its sum of squares and its largest value: a warp holds up to 40 of bf16 (us of 78000 x 1280 with a residual:
// block 142, warp 123; of 130000 x 768: 140, 111), 24 where pieces have four values.  Otherwise of bf16 up to 16 (forward at 768 channels: block 126, warp 137; backward 146, 150), of float32 24 (backward at 512: block
// 142, warp 124).
constexpr int MOST_EIGHT = 40, MOST_BF16 = 16, MOST_F32 = 24;
// How a row is held: pieces of `vec` values, `ch` of them a thread, teams of `threads` (0: the kernels above, which read a row several times).
struct Shape { int vec, ch, threads; bool block; };

// Every operand is (address, stride of rows in values, size of a value).
struct Rows { const void* p; int64_t stride; int size; };
// most: how many values a thread of a warp holds at most; beyond, a block holds the row, 8 values a thread: up to 8192 channels in pieces of four or eight values, up to 4096 in single ones (the threads that
// a block has), in either type; above that none.
template <int N> Shape shape_of(const Rows (&all)[N], int C, int size, int most) {
  auto fits = [&](int v) {
    if (C % v) return false;
    for (const Rows& o : all)
      if (o.p && (o.stride % v || reinterpret_cast<uintptr_t>(o.p) % (v * o.size))) return false;
    return true;
  };
  // 16 bytes a piece; of bf16 8 below 256 channels, where lanes would stay idle (260000 x 384, with a residual: 16 bytes 128 us forward and 122 into 8 bits, 8 bytes 140 and 131)
  const int vec = size == 2 && C >= 256 && fits(8) ? 8 : fits(4) ? 4 : 1;
  const int ch = (C + 32 * vec - 1) / (32 * vec);
  most = vec == 1 ? 8 : vec == 4 ? std::min(most, 24) : most;
  if (ch * vec <= most) return {vec, vec == 1 ? (ch + 3) / 4 * 4 : ch, 32, false};
  const int per = 8 / vec, threads = ((C + 7) / 8 + 31) / 32 * 32;
  if (threads <= (vec == 1 ? BLOCK_MOST<1> : BLOCK_MOST<4>)) return {vec, per, threads, true};
  return {0, 0, 0, false};
}

// Calls f with the pieces' width, their number a thread, and whether a block holds a row, as constants.
template <typename T, typename F> int with(const Shape& s, const F& f) {
#define FOVI_ROWS(V, N, B) if (s.vec == V && s.ch == N && s.block == B) return f(std::integral_constant<int, V>(), std::integral_constant<int, N>(), std::bool_constant<B>())
  if constexpr (sizeof(T) == 2) {
    FOVI_ROWS(8, 1, true); FOVI_ROWS(8, 1, false); FOVI_ROWS(8, 2, false); FOVI_ROWS(8, 3, false);
    FOVI_ROWS(8, 4, false); FOVI_ROWS(8, 5, false);
  }
  FOVI_ROWS(4, 1, false); FOVI_ROWS(4, 2, false); FOVI_ROWS(4, 3, false); FOVI_ROWS(4, 4, false); FOVI_ROWS(4, 5, false); FOVI_ROWS(4, 6, false); FOVI_ROWS(4, 2, true);
  FOVI_ROWS(1, 4, false); FOVI_ROWS(1, 8, false); FOVI_ROWS(1, 8, true);
#undef FOVI_ROWS
  return FOVI_ERR_UNSUPPORTED;
}

template <typename T, int FORM> int rows_forward(const RmsArgs& a, const Shape& s, cudaStream_t st) {
  return with<T>(s, [&](auto vec, auto ch, auto block) {
    auto go = [&](auto kernel, std::atomic<int>* known) {
      const int threads = s.block ? s.threads : 256;
      const int64_t want = s.block ? a.rows : (a.rows + 7) / 8;
      kernel<<<(int)std::min(want, resident(kernel, threads, 0, known[threads / 32])), threads, 0, st>>>(a);
      return fovi::after_launch("rms_norm_rows_kernel");
    };
    static std::atomic<int> known[2][33];
    if constexpr (FORM != ROWS) {
      if (a.res) return go(rms_norm_rows_kernel<T, decltype(vec)::value, decltype(ch)::value, decltype(block)::value, true, FORM>, known[1]);
    }
    return go(rms_norm_rows_kernel<T, decltype(vec)::value, decltype(ch)::value, decltype(block)::value, false, FORM>, known[0]);
  });
}

constexpr int GRAD_BLOCKS = 1184;          // most parts of dw: eight for each of 148 SMs
int strips_of(int64_t rows) { return (int)(rows < 512 ? (rows + 15) / 16 : 64); }

template <typename T, bool NORM> int forward(const RmsArgs& a, cudaStream_t st) {
  const int size = sizeof(T);
  const Shape s = shape_of<5>({{a.x, a.x_stride, size}, {a.res, a.r_stride, size}, {a.total, a.C, size}, {a.y, a.C, size}, {a.q, a.q_stride, 1}}, a.C, size, a.q ? MOST_EIGHT : size == 2 ? MOST_BF16 : MOST_F32);
  if (s.threads) {
    if constexpr (!NORM) return rows_forward<T, ROWS>(a, s, st);
    else return a.q ? rows_forward<T, EIGHT>(a, s, st) : rows_forward<T, PLAIN>(a, s, st);
  }
  const int grid = (int)std::min<int64_t>(a.rows, fovi::sm_count() * 8);
  rms_norm_kernel<T, NORM><<<grid, GEN_THREADS, 0, st>>>(a);
  return fovi::after_launch("rms_norm_kernel");
}

template <typename T> int backward(const RmsGradArgs& a, float* dw, cudaStream_t st) {
  const int size = sizeof(T);
  const Shape s = shape_of<4>({{a.t, a.t_stride, size}, {a.dy, a.dy_stride, size}, {a.dt, a.dt_stride, size}, {a.dx, a.C, size}}, a.C, size, size == 2 ? MOST_BF16 : MOST_F32);
  int parts = strips_of(a.rows);
  if (s.threads) {
    const int rc = with<T>(s, [&](auto vec, auto ch, auto block) {
      static std::atomic<int> known[33];
      auto kernel = rms_norm_grad_rows_kernel<T, decltype(vec)::value, decltype(ch)::value, decltype(block)::value>;
      const int threads = s.block ? s.threads : 256;
      const size_t smem = s.block ? 0 : a.C * sizeof(float);
      const int64_t want = s.block ? a.rows : (a.rows + 7) / 8;
      parts = (int)std::min({want, resident(kernel, threads, smem, known[threads / 32]), (int64_t)GRAD_BLOCKS});
      kernel<<<parts, threads, smem, st>>>(a);
      return fovi::after_launch("rms_norm_grad_rows_kernel");
    });
    if (rc || !dw) return rc;
  } else {
    if (a.dx) {
      const int grid = (int)std::min<int64_t>(a.rows, fovi::sm_count() * 8);
      rms_norm_dx_kernel<T><<<grid, GEN_THREADS, 0, st>>>(a);
      const int rc = fovi::after_launch("rms_norm_dx_kernel");
      if (rc) return rc;
    }
    if (!dw) return FOVI_OK;
    rms_norm_dw_kernel<T><<<dim3((a.C + STRIP_COLS - 1) / STRIP_COLS, parts), STRIP_COLS, 0, st>>>(a, parts);
    const int rc = fovi::after_launch("rms_norm_dw_kernel");
    if (rc) return rc;
  }
  rms_norm_join_kernel<<<(a.C + 31) / 32, 1024, 0, st>>>(a.part, parts, a.C, dw);
  return fovi::after_launch("rms_norm_join_kernel");
}

}  // namespace

extern "C" int fovi_rms_norm_forward(const void* x, int dtype, int64_t rows, int C, int64_t x_stride, const void* residual, int64_t residual_stride, const float* weight,
                                     float eps, void* total, void* y, int8_t* q, int64_t q_stride, float* scale, float* rstd, void* stream) {
  if (rows < 0 || C < 1 || C > MOST_CHANNELS || x_stride < 0 || residual_stride < 0 || !(eps >= 0.f) || !fovi::valid_dtype(dtype)) return FOVI_ERR_INVALID_ARGUMENT;
  if (rows == 0) return FOVI_OK;
  if (!x || (y != nullptr) == (q != nullptr) || (q && (!scale || q_stride < C)) || (residual != nullptr) != (total != nullptr)) return FOVI_ERR_INVALID_ARGUMENT;
  const RmsArgs a{x, residual, rows, C, x_stride, residual_stride, weight, eps, total, y, q, q_stride, scale, rstd};
  auto st = reinterpret_cast<cudaStream_t>(stream);
  return dtype == FOVI_BF16 ? forward<__nv_bfloat16, true>(a, st) : forward<float, true>(a, st);
}

extern "C" int fovi_quantize_rows(const void* x, int dtype, int64_t rows, int C, int64_t x_stride, int8_t* q, int64_t q_stride, float* scale, void* stream) {
  if (rows < 0 || C < 1 || C > MOST_CHANNELS || x_stride < 0 || q_stride < C || !fovi::valid_dtype(dtype)) return FOVI_ERR_INVALID_ARGUMENT;
  if (rows == 0) return FOVI_OK;
  if (!x || !q || !scale) return FOVI_ERR_INVALID_ARGUMENT;
  const RmsArgs a{x, nullptr, rows, C, x_stride, 0, nullptr, 0.f, nullptr, nullptr, q, q_stride, scale, nullptr};
  auto st = reinterpret_cast<cudaStream_t>(stream);
  return dtype == FOVI_BF16 ? forward<__nv_bfloat16, false>(a, st) : forward<float, false>(a, st);
}

extern "C" int64_t fovi_rms_norm_workspace_bytes(int64_t rows, int C) {
  if (rows < 0 || C < 1 || C > MOST_CHANNELS) return -1;
  return std::max<int64_t>(std::min<int64_t>(rows, GRAD_BLOCKS), strips_of(rows)) * C * 4;
}

extern "C" int fovi_rms_norm_backward(const void* t, int dtype, int64_t rows, int C, int64_t t_stride, const void* dy, int64_t dy_stride, const void* dt, int64_t dt_stride,
                                      const float* weight, const float* rstd, void* dx, float* dweight, void* work, int64_t work_bytes, void* stream) {
  if (rows < 0 || C < 1 || C > MOST_CHANNELS || t_stride < 0 || dy_stride < 0 || dt_stride < 0 || !fovi::valid_dtype(dtype)) return FOVI_ERR_INVALID_ARGUMENT;
  auto st = reinterpret_cast<cudaStream_t>(stream);
  if (rows == 0) {
    if (dweight) FOVI_CUDA(cudaMemsetAsync(dweight, 0, (size_t)C * 4, st));
    return FOVI_OK;
  }
  if (!t || !dy || !rstd) return FOVI_ERR_INVALID_ARGUMENT;
  if (dweight && (!work || work_bytes < fovi_rms_norm_workspace_bytes(rows, C))) return FOVI_ERR_INVALID_ARGUMENT;
  const RmsGradArgs a{t, dy, dt, rows, C, t_stride, dy_stride, dt_stride, weight, rstd, dx, dweight ? static_cast<float*>(work) : nullptr};
  return dtype == FOVI_BF16 ? backward<__nv_bfloat16>(a, dweight, st) : backward<float>(a, dweight, st);
}
