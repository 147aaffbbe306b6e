// Layer norm over the last axis of [rows, C], and its gradients:
//   y  = (x - mean) * rstd * w + b          mean, var = mean((x - mean)^2) of the row, rstd = 1 / sqrt(var + eps)
//   dx = rstd * (g - mean(g) - xh * mean(g * xh))          g = dy * w, xh = (x - mean) * rstd
//   dw = sum over rows of dy * xh,   db = sum over rows of dy
// Sums and statistics are float32; results are rounded once, to their tensor's type.  The variance is taken about the row's own mean (two passes over
// values that are already on the chip), so a large common offset does not cost digits.
#include <algorithm>

#include <cuda_bf16.h>

#include "common.cuh"
#include "rows.cuh"

namespace {

constexpr int GEN_THREADS = 256;
constexpr int STRIP_COLS = 128;      // columns of a CTA of the weight-gradient pass

__device__ __forceinline__ float block_sum(float v, float* red) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.f;
  for (int i = 0; i < GEN_THREADS / 32; ++i) t += red[i];
  return t;
}

// One CTA per row, any C.
template <typename TX, typename TY>
__global__ void __launch_bounds__(GEN_THREADS) layer_norm_kernel(const TX* x, int64_t rows, int C, int64_t stride, const float* w, const float* b, float eps, TY* y,
                                                                 float2* stats) {
  __shared__ float red[GEN_THREADS / 32];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const TX* xr = x + r * stride;
    float s = 0.f;
    for (int c = threadIdx.x; c < C; c += GEN_THREADS) s += ld_as_float(xr + c);
    const float mean = block_sum(s, red) / C;
    s = 0.f;
    for (int c = threadIdx.x; c < C; c += GEN_THREADS) { const float d = ld_as_float(xr + c) - mean; s += d * d; }
    const float rstd = 1.f / sqrtf(block_sum(s, red) / C + eps);
    if (stats && threadIdx.x == 0) stats[r] = make_float2(mean, rstd);
    for (int c = threadIdx.x; c < C; c += GEN_THREADS)
      y[r * C + c] = from_float<TY>((ld_as_float(xr + c) - mean) * rstd * (w ? __ldg(w + c) : 1.f) + (b ? __ldg(b + c) : 0.f));
  }
}

template <typename TX, typename TY>
__global__ void __launch_bounds__(GEN_THREADS) layer_norm_dx_kernel(const TX* x, int64_t rows, int C, int64_t stride, const TY* dy, int64_t dy_stride, const float* w,
                                                                    const float2* stats, TX* dx) {
  __shared__ float red[GEN_THREADS / 32];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const float2 st = __ldg(stats + r);
    float sg = 0.f, sgx = 0.f;
    for (int c = threadIdx.x; c < C; c += GEN_THREADS) {
      const float g = ld_as_float(dy + r * dy_stride + c) * (w ? __ldg(w + c) : 1.f);
      sg += g;
      sgx += g * ((ld_as_float(x + r * stride + c) - st.x) * st.y);
    }
    sg = block_sum(sg, red) / C;
    sgx = block_sum(sgx, red) / C;
    for (int c = threadIdx.x; c < C; c += GEN_THREADS) {
      const float g = ld_as_float(dy + r * dy_stride + c) * (w ? __ldg(w + c) : 1.f), xh = (ld_as_float(x + r * stride + c) - st.x) * st.y;
      dx[r * C + c] = from_float<TX>(st.y * (g - sg - xh * sgx));
    }
  }
}

// A thread per column and strip of rows: the strip's part of both sums, [strip][2][C].
template <typename TX, typename TY>
__global__ void __launch_bounds__(STRIP_COLS) layer_norm_dw_kernel(const TX* x, int64_t rows, int C, int64_t stride, const TY* dy, int64_t dy_stride, const float2* stats,
                                                                   float* part, int strips) {
  const int c = blockIdx.x * STRIP_COLS + threadIdx.x;
  if (c >= C) return;
  float sw = 0.f, sb = 0.f;
  for (int64_t r = blockIdx.y; r < rows; r += strips) {
    const float2 st = __ldg(stats + r);
    const float g = ld_as_float(dy + r * dy_stride + c);
    sw += g * ((ld_as_float(x + r * stride + c) - st.x) * st.y);
    sb += g;
  }
  part[((size_t)blockIdx.y * 2) * C + c] = sw;
  part[((size_t)blockIdx.y * 2 + 1) * C + c] = sb;
}

// The parts of dw and db added in a fixed order, the same bits every time: a block takes 32 of the 2C columns, 32 warps every 32nd part.
__global__ void __launch_bounds__(1024) layer_norm_join_kernel(const float* part, int parts, int C, float* dw, float* db) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < 2 * C)
    for (int p = w; p < parts; p += 32) s += part[(size_t)p * 2 * C + c];
  red[w][lane] = s;
  __syncthreads();
  if (w || c >= 2 * C) return;
  s = 0.f;
  for (int i = 0; i < 32; ++i) s += red[i][lane];
  float* to = c < C ? dw : db;
  if (to) to[c < C ? c : c - C] = s;
}

// ------------------------------------------------------------------------------------------------------------ rows in registers
// A row is held in registers by a team of threads, a warp or (rows too long for one) a block, each with CH pieces of VEC values; the next row's loads are issued before this row's
// sums, so that every warp has two rows in flight.  One pass over memory in both directions: the backward kernel reads x and dy once, writes dx, and keeps every column's
// part of dw and db in registers over all rows of its team.  What bounds it is memory, at the rate at which the warps that fit the registers keep loads on the way: 263168 x 384 bf16
// forward 76 us (5.3 TB/s), backward 135 (4.5); 200000 x 384 float32 106 (5.8) and 152 (6.0); 80000 x 1280 bf16 86 (4.8) and 158 (3.9).  Two rows a team at a time were slower
// (126 and 145 us at the first size).  Rows of single values (odd C) are bound by their instructions: 100000 x 517 bf16 107 and 218 us (1.9 and 1.4 TB/s).
template <typename TX, typename TY, int VEC, int CH, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? BLOCK_MOST<VEC> : 256, !BLOCK && sizeof(TX) == 2 && CH * VEC <= 12 ? 4 : 0)
layer_norm_rows_kernel(const TX* __restrict__ x, int64_t rows, int C, int64_t stride, const float* __restrict__ w,
                                                                             const float* __restrict__ b, float eps, TY* __restrict__ y, float2* __restrict__ stats) {
  constexpr int E = CH * VEC, H = VEC > 1 ? VEC / 2 : 1;       // pairs of a piece; single values pair up over two pieces
  constexpr int STEP = VEC > 1 ? 1 : 2;                        // pieces of a step
  __shared__ float2 part[2][32];
  const Team<VEC, BLOCK> t;
  Pairs<E> wv, bv;
  Piece<TX, VEC> next[CH] = {};                                // pieces behind the row's end stay zeros
  int pieces = 0;
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    pieces += t.first + k * t.pitch < C;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int c = t.first + k * t.pitch + i;
      *wv.at(k * VEC + i) = w && c < C ? __ldg(w + c) : 1.f;
      *bv.at(k * VEC + i) = b && c < C ? __ldg(b + c) : 0.f;
    }
  }
  auto fetch = [&](int64_t r) {
#pragma unroll
    for (int k = 0; k < CH; ++k)
      if (k < pieces) next[k] = load_piece<TX, VEC>(x + r * stride + t.first + k * t.pitch);
  };
  if (t.row < rows) fetch(t.row);
  const float n = BLOCK ? warp_sum((float)(pieces * VEC)) : (float)C, inv_n = 1.f / fmaxf(n, 1.f), inv = 1.f / C;
  int flip = 0;
  for (int64_t r = t.row; r < rows; r += t.step, flip ^= 1) {
    Pairs<E> v;
    float2 s2 = both(0.f);
#pragma unroll
    for (int k = 0; k < CH; ++k) widen<TX, VEC>(next[k], v.at(k * VEC));
#pragma unroll
    for (int i = 0; i < E / 2; ++i) s2 = add2(s2, v.v[i]);
    if (r + t.step < rows) fetch(r + t.step);
    // mean and sum of squares about it: of the warp's values, then (block) of all warps' by the parallel form of the same
    float mean = warp_sum(s2.x + s2.y) * inv_n;
    s2 = both(0.f);
#pragma unroll
    for (int k = 0; k < CH; k += STEP) {
      if (k < pieces) {
#pragma unroll
        for (int i = k * VEC / 2; i < k * VEC / 2 + H; ++i) {
          v.v[i] = add2(v.v[i], both(-mean));
          if (STEP == 2 && k + 1 >= pieces) v.v[i].y = 0.f;
          s2 = fma2(v.v[i], v.v[i], s2);
        }
      }
    }
    float q = warp_sum(s2.x + s2.y), shift = 0.f;
    if (BLOCK) {          // a lane per warp: its mean, its sum of squares; how many values it holds follows from the row's length
      if ((threadIdx.x & 31) == 0) part[flip][t.warp] = make_float2(mean, q);
      __syncthreads();    // (two sets of parts: a warp that is ahead writes the other one)
      const int lane = threadIdx.x & 31;
      const float2 p = lane < t.warps ? part[flip][lane] : make_float2(0.f, 0.f);
      float held = 0.f;
#pragma unroll
      for (int k = 0; k < CH; ++k) held += (float)min(max(C - (lane * 32 * VEC + k * t.pitch), 0), 32 * VEC);
      if (lane >= t.warps) held = 0.f;
      const float all = warp_sum(held * p.x) * inv, d = p.x - all;
      q = warp_sum(held > 0.f ? fmaf(held * d, d, p.y) : 0.f);
      shift = mean - all;
      mean = all;
    }
    const float rstd = rsqrtf(fmaf(q, inv, eps));
    if (stats && (BLOCK ? threadIdx.x : threadIdx.x & 31) == 0) stats[r] = make_float2(mean, rstd);
#pragma unroll
    for (int k = 0; k < CH; k += STEP) {
      if (k < pieces) {
        Pairs<VEC * STEP> o;
#pragma unroll
        for (int i = 0; i < H; ++i) {
          const int e = k * VEC / 2 + i;
          o.v[i] = fma2(mul2(BLOCK ? add2(v.v[e], both(shift)) : v.v[e], both(rstd)), wv.v[e], bv.v[e]);
        }
        store_piece<TY, VEC>(y + r * C + t.first + k * t.pitch, o.at(0));
        if (STEP == 2 && k + 1 < pieces) store_piece<TY, VEC>(y + r * C + t.first + (k + 1) * t.pitch, o.at(1));
      }
    }
  }
}

template <typename TX, typename TY, int VEC, int CH, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? BLOCK_MOST<VEC> : 256, BLOCK ? 1 : CH * VEC <= 8 ? 3 : 2)
layer_norm_grad_rows_kernel(const TX* __restrict__ x, int64_t rows, int C, int64_t stride, const TY* __restrict__ dy, int64_t dy_stride, const float* __restrict__ w,
                            const float2* __restrict__ stats, TX* __restrict__ dx, float* __restrict__ part) {
  constexpr int E = CH * VEC, H = VEC > 1 ? VEC / 2 : 1, STEP = VEC > 1 ? 1 : 2;
  __shared__ float2 sums[2][32];
  extern __shared__ float4 joined4[];        // warp teams: the weights (in shared memory: their registers are a third block's), then the warps' parts, [2][C]
  float* joined = reinterpret_cast<float*>(joined4);
  const Team<VEC, BLOCK> t;
  Pairs<BLOCK ? E : 2> wv;
  Pairs<E> aw, ab;
  Piece<TX, VEC> nx[CH] = {};
  Piece<TY, VEC> ng[CH] = {};
  int pieces = 0;
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    pieces += t.first + k * t.pitch < C;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int c = t.first + k * t.pitch + i;
      if (BLOCK) *wv.at(BLOCK ? k * VEC + i : 0) = w && c < C ? __ldg(w + c) : 1.f;
      *aw.at(k * VEC + i) = *ab.at(k * VEC + i) = 0.f;
    }
  }
  if (!BLOCK) {
    for (int c = threadIdx.x; c < C; c += blockDim.x) joined[c] = w ? __ldg(w + c) : 1.f;
    __syncthreads();
  }
  float2 ns = make_float2(0.f, 0.f);
  auto fetch = [&](int64_t r) {
    ns = __ldg(stats + r);
#pragma unroll
    for (int k = 0; k < CH; ++k)
      if (k < pieces) {
        nx[k] = load_piece<TX, VEC>(x + r * stride + t.first + k * t.pitch);
        ng[k] = load_piece<TY, VEC>(dy + r * dy_stride + t.first + k * t.pitch);
      }
  };
  if (t.row < rows) fetch(t.row);
  const float inv = 1.f / C;
  int flip = 0;
  for (int64_t r = t.row; r < rows; r += t.step, flip ^= 1) {
    const float rstd = ns.y;
    Pairs<E> xh, g;
    float2 sg = both(0.f), sx = both(0.f);
#pragma unroll
    for (int k = 0; k < CH; ++k) { widen<TX, VEC>(nx[k], xh.at(k * VEC)); widen<TY, VEC>(ng[k], g.at(k * VEC)); }
#pragma unroll
    for (int k = 0; k < CH; k += STEP) {
      if (k < pieces) {                     // (a single value without a second: its gradient is zero, and so is all that it adds)
#pragma unroll
        for (int i = 0; i < H; ++i) {
          const int e = k * VEC / 2 + i;
          float2 we;
          if (BLOCK) we = wv.v[BLOCK ? e : 0];
          else if (VEC > 1) we = *reinterpret_cast<const float2*>(joined + t.first + k * t.pitch + 2 * i);
          else we = make_float2(joined[t.first + k * t.pitch], k + 1 < pieces ? joined[t.first + (k + 1) * t.pitch] : 0.f);
          xh.v[e] = mul2(add2(xh.v[e], both(-ns.x)), both(rstd));
          aw.v[e] = fma2(g.v[e], xh.v[e], aw.v[e]);
          ab.v[e] = add2(ab.v[e], g.v[e]);
          g.v[e] = mul2(g.v[e], we);
          sg = add2(sg, g.v[e]);
          sx = fma2(g.v[e], xh.v[e], sx);
        }
      }
    }
    if (r + t.step < rows) fetch(r + t.step);
    float mg = warp_sum(sg.x + sg.y), mx = warp_sum(sx.x + sx.y);
    if (BLOCK) {
      if ((threadIdx.x & 31) == 0) sums[flip][t.warp] = make_float2(mg, mx);
      __syncthreads();
      const float2 p = (int)(threadIdx.x & 31) < t.warps ? sums[flip][threadIdx.x & 31] : make_float2(0.f, 0.f);
      mg = warp_sum(p.x);
      mx = warp_sum(p.y);
    }
    mg *= inv;
    mx *= inv;
    if (dx) {
#pragma unroll
      for (int k = 0; k < CH; k += STEP) {
        if (k < pieces) {
          Pairs<VEC * STEP> o;
#pragma unroll
          for (int i = 0; i < H; ++i) {
            const int e = k * VEC / 2 + i;
            o.v[i] = mul2(fma2(xh.v[e], both(-mx), add2(g.v[e], both(-mg))), both(rstd));
          }
          store_piece<TX, VEC>(dx + r * C + t.first + k * t.pitch, o.at(0));
          if (STEP == 2 && k + 1 < pieces) store_piece<TX, VEC>(dx + r * C + t.first + (k + 1) * t.pitch, o.at(1));
        }
      }
    }
  }
  if (!part) return;
  float* mine = part + (size_t)blockIdx.x * 2 * C;
  if (!BLOCK) __syncthreads();             // the weights have been read
  if (!BLOCK) {                            // the warps' parts one after another: a fixed order
    for (int u = 0; u < t.warps; ++u) {
      if (t.warp == u) {
#pragma unroll
        for (int k = 0; k < CH; ++k)
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const int c = t.first + k * t.pitch + i;
            if (c < C) {
              joined[c] = (u ? joined[c] : 0.f) + *aw.at(k * VEC + i);
              joined[C + c] = (u ? joined[C + c] : 0.f) + *ab.at(k * VEC + i);
            }
          }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < 2 * C; c += blockDim.x) mine[c] = joined[c];
  } else {
#pragma unroll
    for (int k = 0; k < CH; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int c = t.first + k * t.pitch + i;
        if (c < C) { mine[c] = *aw.at(k * VEC + i); mine[C + c] = *ab.at(k * VEC + i); }
      }
  }
}

// How a row is held: pieces of `vec` values, `ch` of them a thread, teams of `threads` (0: the kernels above, which read a row several times).
struct Shape { int vec, ch, threads; bool block; };
Shape shape_of(const void* x, int64_t x_stride, int xs, const void* y, int64_t y_stride, int ys, int C) {
  auto fits = [&](int v) {
    return C % v == 0 && x_stride % v == 0 && y_stride % v == 0 && (reinterpret_cast<uintptr_t>(x) % (v * xs)) == 0 && (reinterpret_cast<uintptr_t>(y) % (v * ys)) == 0;
  };
  // VEC 8 is for bf16 on both sides, 16 bytes, from 512 channels on: below, lanes stay idle (forward at 384 channels 84 us in place of 75, backward 142 of 135); at 512 and 768 the two are
  // equal to 2 %, and from 1024 on 16 bytes are the faster ones (backward at 1280 channels 158 us in place of 185).
  const bool wide = xs == 4 || ys == 4;
  const int vec = !wide && C >= 512 && fits(8) ? 8 : fits(4) ? 4 : 1;
  // A warp holds up to 24 values a thread of bf16, 12 of float32 or one by one; beyond, its registers would leave too few warps on an SM.
  int ch = (C + 32 * vec - 1) / (32 * vec);
  if (vec == 1) ch = (ch + 3) / 4 * 4;
  if (ch * vec <= (wide || vec == 1 ? 12 : 24)) return {vec, ch, 32, false};
  const int per = vec == 8 ? 1 : vec == 4 ? 2 : 8;             // a block: 8 values a thread
  const int threads = ((C + per * vec - 1) / (per * vec) + 31) / 32 * 32;
  if (threads <= (vec == 1 ? BLOCK_MOST<1> : BLOCK_MOST<4>)) return {vec, per, threads, true};
  return {0, 0, 0, false};
}

// Blocks of the backward kernel, a part of dw and db each: as many as the SMs hold at once by its registers, three an SM for teams of a warp with up to 8 values a thread and two beyond, about
// 640 threads an SM for teams of a block.  Half as many, this many, twice as many (us): 263168 x 384 bf16 207, 135, 146; 80000 x 1280 bf16 249, 159, 169; 200000 x 384 float32 196, 152, 163;
// 100000 x 1024 bf16, whose blocks of 128 threads the limit of 592 cuts short, 299, 183, 131.
constexpr int GRAD_BLOCKS = 592;         // most parts: four for each of 148 SMs
int grad_blocks(const Shape& s, int64_t rows) {
  const int64_t want = s.block ? rows : (rows + 7) / 8, sms = fovi::sm_count();
  const int64_t most = s.block ? std::max(sms, sms * 640 / s.threads) : s.ch * s.vec <= 8 ? 3 * sms : 2 * sms;
  return (int)std::min({want, most, (int64_t)GRAD_BLOCKS});
}

template <typename TX, typename TY> struct Run {
  const void* x; int64_t rows; int C; int64_t stride; const float* w; const float* b; float eps; void* y; float* stats;
  const void* dy; int64_t dy_stride; void* dx; float* part; cudaStream_t st;
  template <int VEC, int CH, bool BLOCK> int go(const Shape& s, bool backward) const {
    const int threads = BLOCK ? s.threads : 256;
    if (!backward) {
      auto k = layer_norm_rows_kernel<TX, TY, VEC, CH, BLOCK>;
      const int64_t want = BLOCK ? rows : (rows + 7) / 8;
      static std::atomic<int> known[33];
      k<<<(int)std::min(want, resident(k, threads, 0, known[threads / 32])), threads, 0, st>>>((const TX*)x, rows, C, stride, w, b, eps, (TY*)y, (float2*)stats);
      return fovi::after_launch("layer_norm_rows_kernel");
    }
    auto k = layer_norm_grad_rows_kernel<TX, TY, VEC, CH, BLOCK>;
    k<<<grad_blocks(s, rows), threads, BLOCK ? 0 : 2 * C * sizeof(float), st>>>((const TX*)x, rows, C, stride, (const TY*)dy, dy_stride, w, (const float2*)stats, (TX*)dx, part);
    return fovi::after_launch("layer_norm_grad_rows_kernel");
  }
  template <int VEC, int MOST, int STEP = 1, int CH = STEP> int warp(const Shape& s, bool backward) const {
    if constexpr (CH * VEC <= MOST) return s.ch == CH ? go<VEC, CH, false>(s, backward) : warp<VEC, MOST, STEP, CH + STEP>(s, backward);
    return FOVI_ERR_UNSUPPORTED;
  }
  int operator()(const Shape& s, bool backward) const {
    if (s.block) {
      if constexpr (sizeof(TX) == 2 && sizeof(TY) == 2) {
        if (s.vec == 8) return go<8, 1, true>(s, backward);
      }
      return s.vec == 4 ? go<4, 2, true>(s, backward) : go<1, 8, true>(s, backward);
    }
    if constexpr (sizeof(TX) == 2 && sizeof(TY) == 2) {
      if (s.vec == 8) return warp<8, 24>(s, backward);
      if (s.vec == 4) return warp<4, 24>(s, backward);
    }
    return s.vec == 4 ? warp<4, 12>(s, backward) : warp<1, 12, 4>(s, backward);
  }
};

// ------------------------------------------------------------------------------------------------------------ host
int strips_of(int64_t rows) { return (int)(rows < 512 ? (rows + 15) / 16 : 64); }

template <typename TX, typename TY>
int forward(const void* x, int64_t rows, int C, int64_t stride, const float* w, const float* b, float eps, void* y, float* stats, cudaStream_t st) {
  const Shape s = shape_of(x, stride, sizeof(TX), y, C, sizeof(TY), C);
  if (s.threads) return Run<TX, TY>{x, rows, C, stride, w, b, eps, y, stats, nullptr, 0, nullptr, nullptr, st}(s, false);
  const int grid = (int)std::min<int64_t>(rows, fovi::sm_count() * 8);
  layer_norm_kernel<TX, TY><<<grid, GEN_THREADS, 0, st>>>((const TX*)x, rows, C, stride, w, b, eps, (TY*)y, (float2*)stats);
  return fovi::after_launch("layer_norm_kernel");
}

template <typename TX, typename TY>
int backward(const void* x, int64_t rows, int C, int64_t stride, const void* dy, int64_t dy_stride, const float* w, const float* stats, void* dx, float* dw, float* db,
             float* work, cudaStream_t st) {
  Shape s = shape_of(x, stride, sizeof(TX), dy, dy_stride, sizeof(TY), C);
  if (s.threads && dx && (reinterpret_cast<uintptr_t>(dx) % (s.vec * sizeof(TX)))) s.threads = 0;
  int strips = strips_of(rows);
  if (s.threads) {
    const int rc = Run<TX, TY>{x, rows, C, stride, w, nullptr, 0.f, nullptr, const_cast<float*>(stats), dy, dy_stride, dx, dw || db ? work : nullptr, st}(s, true);
    if (rc || !(dw || db)) return rc;
    strips = grad_blocks(s, rows);
  } else {
    if (dx) {
      const int grid = (int)std::min<int64_t>(rows, fovi::sm_count() * 8);
      layer_norm_dx_kernel<TX, TY><<<grid, GEN_THREADS, 0, st>>>((const TX*)x, rows, C, stride, (const TY*)dy, dy_stride, w, (const float2*)stats, (TX*)dx);
      const int rc = fovi::after_launch("layer_norm_dx_kernel");
      if (rc) return rc;
    }
    if (!dw && !db) return FOVI_OK;
    const dim3 grid((C + STRIP_COLS - 1) / STRIP_COLS, strips);
    layer_norm_dw_kernel<TX, TY><<<grid, STRIP_COLS, 0, st>>>((const TX*)x, rows, C, stride, (const TY*)dy, dy_stride, (const float2*)stats, work, strips);
    const int rc = fovi::after_launch("layer_norm_dw_kernel");
    if (rc) return rc;
  }
  layer_norm_join_kernel<<<(2 * C + 31) / 32, 1024, 0, st>>>(work, strips, C, dw, db);
  return fovi::after_launch("layer_norm_join_kernel");
}

}  // namespace

extern "C" int64_t fovi_layer_norm_workspace_bytes(int64_t rows, int C) {
  if (rows < 0 || C < 1) return -1;
  return std::max<int64_t>(std::min<int64_t>(rows, GRAD_BLOCKS), strips_of(rows)) * 2 * C * 4;
}

extern "C" int fovi_layer_norm_forward(const void* x, int x_dtype, int64_t rows, int C, int64_t x_stride, const float* weight, const float* bias, float eps, void* y,
                                       int y_dtype, float* stats, void* stream) {
  if (rows < 0 || C < 1 || x_stride < 0 || !(eps >= 0.f) || !fovi::valid_dtype(x_dtype) || !fovi::valid_dtype(y_dtype)) return FOVI_ERR_INVALID_ARGUMENT;
  if (rows == 0) return FOVI_OK;
  if (!x || !y) return FOVI_ERR_INVALID_ARGUMENT;
  auto st = reinterpret_cast<cudaStream_t>(stream);
  const bool xb = x_dtype == FOVI_BF16, yb = y_dtype == FOVI_BF16;
  if (xb) return yb ? forward<__nv_bfloat16, __nv_bfloat16>(x, rows, C, x_stride, weight, bias, eps, y, stats, st)
                    : forward<__nv_bfloat16, float>(x, rows, C, x_stride, weight, bias, eps, y, stats, st);
  return yb ? forward<float, __nv_bfloat16>(x, rows, C, x_stride, weight, bias, eps, y, stats, st)
            : forward<float, float>(x, rows, C, x_stride, weight, bias, eps, y, stats, st);
}

extern "C" int fovi_layer_norm_backward(const void* x, int x_dtype, int64_t rows, int C, int64_t x_stride, const void* dy, int y_dtype, int64_t dy_stride,
                                        const float* weight, const float* stats, void* dx, float* dweight, float* dbias, void* work, int64_t work_bytes, void* stream) {
  if (rows < 0 || C < 1 || x_stride < 0 || dy_stride < 0 || !fovi::valid_dtype(x_dtype) || !fovi::valid_dtype(y_dtype)) return FOVI_ERR_INVALID_ARGUMENT;
  auto st = reinterpret_cast<cudaStream_t>(stream);
  if (rows == 0) {
    if (dweight) FOVI_CUDA(cudaMemsetAsync(dweight, 0, (size_t)C * 4, st));
    if (dbias) FOVI_CUDA(cudaMemsetAsync(dbias, 0, (size_t)C * 4, st));
    return FOVI_OK;
  }
  if (!x || !dy || !stats) return FOVI_ERR_INVALID_ARGUMENT;
  if ((dweight || dbias) && (!work || work_bytes < fovi_layer_norm_workspace_bytes(rows, C))) return FOVI_ERR_INVALID_ARGUMENT;
  const bool xb = x_dtype == FOVI_BF16, yb = y_dtype == FOVI_BF16;
  float* wk = static_cast<float*>(work);
  if (xb) return yb ? backward<__nv_bfloat16, __nv_bfloat16>(x, rows, C, x_stride, dy, dy_stride, weight, stats, dx, dweight, dbias, wk, st)
                    : backward<__nv_bfloat16, float>(x, rows, C, x_stride, dy, dy_stride, weight, stats, dx, dweight, dbias, wk, st);
  return yb ? backward<float, __nv_bfloat16>(x, rows, C, x_stride, dy, dy_stride, weight, stats, dx, dweight, dbias, wk, st)
            : backward<float, float>(x, rows, C, x_stride, dy, dy_stride, weight, stats, dx, dweight, dbias, wk, st);
}
