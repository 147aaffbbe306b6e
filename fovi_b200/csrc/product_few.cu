// Matrix products of few tokens, 16 a block: y[m, n] = sum over k of x[m, k] w[n, k], bf16 or 8-bit integers.
//
// What bounds them is how fast the weights come: each is used by up to 16 tokens of a block.  A block takes 16 rows of w (GATED: of both matrices) and divides k among its warps in
// turns of 64 bytes a row; a warp's loads are 16 bytes a lane, four lanes side by side in a row, straight into the registers that the matrix instruction (m16n8k16 or m16n8k32: weights
// are its 16 rows, tokens its 8 columns) takes them from.  That an instruction's k then is not consecutive does not matter, since tokens are loaded the same way.
// Two turns' loads are on their way while two are worked on (GATED: one and one, so that three blocks fit an SM and 5120 rows are one round of them).  The warps' sums are joined in shared
// memory in a fixed order, and a thread for each result ends it.
// One token through 1280 x 5120 channels, 39 MB of weights: 13.3 us from memory (3.0 TB/s; 12.8 with h in one part), 8.4 from L2.
// The tensor cores' large instructions (product_tc.cu) have 128 rows: with one token 5120 x 1280 8-bit weights take 8.8 us there, 3.0 to 4.5 here.
#include <algorithm>

#include "product_few.cuh"
#include "tc_common.cuh"

using fovi::FewRows;

namespace {

enum { GATED = 0, LINEAR = 1, SCALED = 2 };
constexpr int ROWS = 16;

struct FewArgs {
  const char *x, *w, *w2; int64_t x_pitch, w_pitch, w2_pitch;        // pitches in bytes
  int64_t rest;                                                      // LINEAR, GATED: bytes from h to its rest
  int m, n, k;                                                       // k in bytes
  const __nv_bfloat16 *bias, *bias2; int act;
  const float *scale, *wscale, *bias_f; int y_f32;
  void* y; int64_t y_pitch;                                          // in values
};

__device__ __forceinline__ void mma_few(float (&d)[4], const uint32_t* a, const uint32_t* b, uint32_t a0, uint32_t a1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a0), "r"(a[1]), "r"(a1), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ void mma_few(int (&d)[4], const uint32_t* a, const uint32_t* b, uint32_t a0, uint32_t a1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a[0]), "r"(a0), "r"(a[1]), "r"(a1), "r"(b[0]), "r"(b[1]));
}
template <bool I8> struct SumT { using type = float; };
template <> struct SumT<true> { using type = int; };

struct Piece16 { uint32_t w[4]; };
// 16 bytes of a row from byte `at` on, of which those behind the row's `end` are zeros whatever lies there.  No branches: the lanes of a warp stay together for the matrix instructions,
// which are the whole warp's (with the loads in branches on a lane's row and column, lanes could reach them apart).  Weights: read once; tokens may come from the launch before: a load
// that stays behind the wait for it.
template <bool WEIGHTS> __device__ __forceinline__ Piece16 load16(const char* row, bool here, int at, int end) {
  Piece16 p;
  const int left = end - at, use = here && left > 0;
  if (WEIGHTS)
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %5, 0;\n mov.b32 %0, 0;\n mov.b32 %1, 0;\n mov.b32 %2, 0;\n mov.b32 %3, 0;\n"
                 " @p ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];\n}\n"
                 : "=&r"(p.w[0]), "=&r"(p.w[1]), "=&r"(p.w[2]), "=&r"(p.w[3]) : "l"(row + at), "r"(use));
  else
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %5, 0;\n mov.b32 %0, 0;\n mov.b32 %1, 0;\n mov.b32 %2, 0;\n mov.b32 %3, 0;\n"
                 " @p ld.global.v4.b32 {%0, %1, %2, %3}, [%4];\n}\n"
                 : "=&r"(p.w[0]), "=&r"(p.w[1]), "=&r"(p.w[2]), "=&r"(p.w[3]) : "l"(row + at), "r"(use) : "memory");
#pragma unroll
  for (int i = 0; i < 4; ++i) p.w[i] &= (uint32_t)((1ull << 8 * min(max(left - 4 * i, 0), 4)) - 1ull);
  return p;
}

template <int EPI, int NT, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, EPI == GATED && WARPS == 8 ? 3 : 1) product_few_kernel(const __grid_constant__ FewArgs a, const int early) {
  constexpr bool I8 = EPI == SCALED, TWO = EPI == GATED;
  constexpr int MATS = TWO ? 2 : 1, COLS = NT * 8, TURNS = TWO ? 1 : 2, PARTS = EPI == LINEAR ? 2 : 1;
  using S = typename SumT<I8>::type;
  __shared__ S part[WARPS][MATS][ROWS][COLS + 2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * ROWS, m0 = blockIdx.y * 16;
  const bool low = n0 + r < a.n, high = n0 + r + 8 < a.n;
  const char *w[MATS][2], *x[NT];
  w[0][0] = a.w + (int64_t)(n0 + r) * a.w_pitch;
  w[0][1] = w[0][0] + 8 * a.w_pitch;
  if (TWO) {
    w[MATS - 1][0] = a.w2 + (int64_t)(n0 + r) * a.w2_pitch;
    w[MATS - 1][1] = w[MATS - 1][0] + 8 * a.w2_pitch;
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) x[j] = a.x + (int64_t)(m0 + 8 * j + r) * a.x_pitch;
  Piece16 wp[2][TURNS][MATS][2], xp[2][TURNS][PARTS][NT];
  constexpr int STEP = WARPS * 64, ROUND = TURNS * STEP;
  const int first = warp * 64, own = t * 16;
  auto weights = [&](int set, int at) {
#pragma unroll
    for (int u = 0; u < TURNS; ++u)
#pragma unroll
      for (int q = 0; q < MATS; ++q) {
        wp[set][u][q][0] = load16<true>(w[q][0], low, at + u * STEP + own, a.k);
        wp[set][u][q][1] = load16<true>(w[q][1], high, at + u * STEP + own, a.k);
      }
  };
  auto tokens = [&](int set, int at) {
#pragma unroll
    for (int u = 0; u < TURNS; ++u)
#pragma unroll
      for (int p = 0; p < PARTS; ++p)
#pragma unroll
        for (int j = 0; j < NT; ++j) xp[set][u][p][j] = load16<false>(x[j] + p * a.rest, m0 + 8 * j + r < a.m, at + u * STEP + own, a.k);
  };
  S d[MATS][NT][4] = {};
  auto products = [&](int set) {
#pragma unroll
    for (int u = 0; u < TURNS; ++u)
#pragma unroll
      for (int q = 0; q < MATS; ++q)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
          for (int p = PARTS - 1; p >= 0; --p) {
            const uint32_t *w0 = wp[set][u][q][0].w, *w1 = wp[set][u][q][1].w, *v = xp[set][u][p][j].w;
            mma_few(d[q][j], w0, v, w1[0], w1[1]);
            mma_few(d[q][j], w0 + 2, v + 2, w1[2], w1[3]);
          }
        }
  };
  // The weights do not come from the launch before: where that is known to be this call's own, they are asked for in front of the wait for it.
  if (early) weights(0, first);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (!early) weights(0, first);
  tokens(0, first);
  for (int at = first; at < a.k; at += 2 * ROUND) {               // (the same turns for all lanes, as the instruction is the warp's)
    weights(1, at + ROUND);
    tokens(1, at + ROUND);
    products(0);
    if (at + ROUND >= a.k) break;
    weights(0, at + 2 * ROUND);
    tokens(0, at + 2 * ROUND);
    products(1);
  }
#pragma unroll
  for (int q = 0; q < MATS; ++q)
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      part[warp][q][r][8 * j + 2 * t] = d[q][j][0];
      part[warp][q][r][8 * j + 2 * t + 1] = d[q][j][1];
      part[warp][q][r + 8][8 * j + 2 * t] = d[q][j][2];
      part[warp][q][r + 8][8 * j + 2 * t + 1] = d[q][j][3];
    }
  __syncthreads();
  for (int e = threadIdx.x; e < ROWS * COLS; e += WARPS * 32) {
    const int i = e % ROWS, col = e / ROWS, m = m0 + col, n = n0 + i;               // neighbouring threads write neighbouring values
    if (m >= a.m || n >= a.n) continue;
    S s[MATS] = {};
#pragma unroll
    for (int v = 0; v < WARPS; ++v)
#pragma unroll
      for (int q = 0; q < MATS; ++q) s[q] += part[v][q][i][col];
    const int64_t at = m * a.y_pitch + n;
    if (EPI == SCALED) {
      const float y = fmaf((float)s[0] * __ldg(a.scale + m), __ldg(a.wscale + n), a.bias_f ? __ldg(a.bias_f + n) : 0.f);
      if (a.y_f32) static_cast<float*>(a.y)[at] = y;
      else static_cast<__nv_bfloat16*>(a.y)[at] = __float2bfloat16_rn(y);
    } else if (EPI == GATED) {
      const float g = s[0] + (a.bias ? __bfloat162float(__ldg(a.bias + n)) : 0.f), u = s[MATS - 1] + (a.bias2 ? __bfloat162float(__ldg(a.bias2 + n)) : 0.f);
      const float p = a.act == fovi::ACT_SILU ? __fdividef(1.f, 1.f + __expf(-g)) : 0.5f * (1.f + erff(g * 0.70710678118654752f));
      const float h = g * p * u, high = fminf(fmaxf(h, -3.38953139e38f), 3.38953139e38f);       // the largest bf16 value: infinity is the rest
      const __nv_bfloat16 part = __float2bfloat16_rn(high);
      static_cast<__nv_bfloat16*>(a.y)[at] = part;
      reinterpret_cast<__nv_bfloat16*>(static_cast<char*>(a.y) + a.rest)[at] = __float2bfloat16_rn(h - __bfloat162float(part));
    } else {
      static_cast<__nv_bfloat16*>(a.y)[at] = __float2bfloat16_rn(s[0] + (a.bias ? __bfloat162float(__ldg(a.bias + n)) : 0.f));
    }
  }
}

// ------------------------------------------------------------------------------------------------------------ float32
// The same with multiply-adds: a block takes 16 rows and 8 tokens; a lane has 16 bytes of two rows (GATED: of each matrix) and their products with the eight tokens, whose values come
// through L1; the four lanes of a row and the warps join their sums in a fixed order.
// 1280 x 3416 channels, 52 MB of weights: one token 28 us, eight 48 (1.9 and 1.1 TB/s): two turns of weights are on their way, and a turn's tokens are eight loads and as many chains of multiply-adds.
struct Few32Args {
  const float *x, *w, *w2; int64_t x_pitch, w_pitch, w2_pitch;
  int m, n, k, act;
  const float *bias, *bias2;
  float* y; int64_t y_pitch;
  int x_vec, w_vec;                // rows start on 16-byte boundaries
};
// Four values of a row from `at` on, of which those behind the row's end are zeros.
__device__ __forceinline__ float4 load4(const float* row, bool here, int at, int end, bool vec, bool stream) {
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  if (here && at < end) {
    if (vec && at + 4 <= end) {
      if (stream) asm volatile("ld.global.nc.L1::no_allocate.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "l"(row + at));
      else asm volatile("ld.global.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "l"(row + at) : "memory");
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (at + i < end) asm volatile("ld.global.f32 %0, [%1];" : "=f"(v[i]) : "l"(row + at + i) : "memory");
    }
  }
  return make_float4(v[0], v[1], v[2], v[3]);
}

template <bool TWO>
__global__ void __launch_bounds__(256) product_few32_kernel(const __grid_constant__ Few32Args a) {
  constexpr int MATS = TWO ? 2 : 1, WARPS = 8, TOK = 8;
  __shared__ float part[WARPS][MATS][ROWS][TOK + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3, n0 = blockIdx.x * ROWS, m0 = blockIdx.y * TOK;
  const bool there[2] = {n0 + r < a.n, n0 + r + 8 < a.n};
  const float* w[MATS][2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    w[0][h] = a.w + (int64_t)(n0 + r + 8 * h) * a.w_pitch;
    if (TWO) w[MATS - 1][h] = a.w2 + (int64_t)(n0 + r + 8 * h) * a.w2_pitch;
  }
  float d[MATS][2][TOK] = {};
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  constexpr int STEP = WARPS * 16, TURNS = 2;           // two turns at a time, the next two on their way
  float4 next[TURNS][MATS][2];
  auto weights = [&](int at) {
#pragma unroll
    for (int u = 0; u < TURNS; ++u)
#pragma unroll
      for (int q = 0; q < MATS; ++q)
#pragma unroll
        for (int h = 0; h < 2; ++h) next[u][q][h] = load4(w[q][h], there[h], at + u * STEP, a.k, a.w_vec, true);
  };
  const float* x = a.x + (int64_t)m0 * a.x_pitch;
  const int first = warp * 16 + 4 * t, tokens = a.m - m0;
  weights(first);
  for (int at = first; at < a.k; at += TURNS * STEP) {
    float4 now[TURNS][MATS][2];
#pragma unroll
    for (int u = 0; u < TURNS; ++u)
#pragma unroll
      for (int q = 0; q < MATS; ++q)
#pragma unroll
        for (int h = 0; h < 2; ++h) now[u][q][h] = next[u][q][h];
    weights(at + TURNS * STEP);
#pragma unroll
    for (int u = 0; u < TURNS; ++u) {
      float4 v[TOK];
#pragma unroll
      for (int m = 0; m < TOK; ++m) v[m] = load4(x + m * a.x_pitch, m < tokens, at + u * STEP, a.k, a.x_vec, false);
#pragma unroll
      for (int m = 0; m < TOK; ++m) {
        if (m > 0 && m >= tokens) break;
#pragma unroll
        for (int q = 0; q < MATS; ++q)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            d[q][h][m] = fmaf(now[u][q][h].w, v[m].w, fmaf(now[u][q][h].z, v[m].z, fmaf(now[u][q][h].y, v[m].y, fmaf(now[u][q][h].x, v[m].x, d[q][h][m]))));
      }
    }
  }
  __syncwarp();
#pragma unroll
  for (int q = 0; q < MATS; ++q)
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int m = 0; m < TOK; ++m) {
        float s = d[q][h][m];
        s += __shfl_xor_sync(0xffffffffu, s, 1);
        s += __shfl_xor_sync(0xffffffffu, s, 2);
        if (t == 0) part[warp][q][r + 8 * h][m] = s;
      }
  __syncthreads();
  if (threadIdx.x >= ROWS * TOK) return;
  const int i = threadIdx.x % ROWS, col = threadIdx.x / ROWS, m = m0 + col, n = n0 + i;
  if (m >= a.m || n >= a.n) return;
  float s[MATS] = {};
#pragma unroll
  for (int v = 0; v < WARPS; ++v)
#pragma unroll
    for (int q = 0; q < MATS; ++q) s[q] += part[v][q][i][col];
  if (a.bias) s[0] += __ldg(a.bias + n);
  if (TWO) {
    if (a.bias2) s[MATS - 1] += __ldg(a.bias2 + n);
    const float g = s[0], p = a.act == fovi::ACT_SILU ? 1.f / (1.f + expf(-g)) : 0.5f * (1.f + erff(g * 0.70710678118654752f));
    s[0] = g * p * s[MATS - 1];
  }
  a.y[m * a.y_pitch + n] = s[0];
}

template <int EPI, int NT, int WARPS> int launch(const FewArgs& a, bool early, cudaStream_t st) {
  FOVI_CUDA(fovi::launch_pdl(product_few_kernel<EPI, NT, WARPS>, dim3((a.n + ROWS - 1) / ROWS, (a.m + 15) / 16), WARPS * 32, 0, st, a, (int)early));
  return fovi::after_launch("product_few_kernel");
}
template <int EPI, int NT> int by_warps(const FewArgs& a, bool early, cudaStream_t st) {
  // Fewer blocks than SMs: more warps each.
  return (a.n + ROWS - 1) / ROWS * ((a.m + 15) / 16) < fovi::sm_count() ? launch<EPI, NT, 16>(a, early, st) : launch<EPI, NT, 8>(a, early, st);
}
template <int EPI> int by_tokens(const FewArgs& a, bool early, cudaStream_t st) {
  return a.m <= 8 ? by_warps<EPI, 1>(a, early, st) : by_warps<EPI, 2>(a, early, st);
}

FewArgs args(const FewRows& x, const FewRows& w, int m, int n, int k, int size) {
  FewArgs a{};
  a.x = static_cast<const char*>(x.p); a.x_pitch = x.pitch * size;
  a.w = static_cast<const char*>(w.p); a.w_pitch = w.pitch * size;
  a.m = m; a.n = n; a.k = k * size;
  return a;
}

}  // namespace

int fovi::few_gated(const FewRows& x, const FewRows& wg, const FewRows& wu, int m, int n, int k, const void* bg, const void* bu, int act, const FewRows& h, cudaStream_t st) {
  FewArgs a = args(x, wg, m, n, k, 2);
  a.w2 = static_cast<const char*>(wu.p); a.w2_pitch = wu.pitch * 2;
  a.bias = static_cast<const __nv_bfloat16*>(bg); a.bias2 = static_cast<const __nv_bfloat16*>(bu); a.act = act;
  a.y = const_cast<void*>(h.p); a.y_pitch = h.pitch; a.rest = m * h.pitch * 2;
  return by_tokens<GATED>(a, false, st);
}

int fovi::few_down(const FewRows& h, const FewRows& w, int m, int n, int k, const void* bias, void* y, cudaStream_t st) {
  FewArgs a = args(h, w, m, n, k, 2);
  a.bias = static_cast<const __nv_bfloat16*>(bias);
  a.rest = m * h.pitch * 2;
  a.y = y; a.y_pitch = n;
  return by_tokens<LINEAR>(a, true, st);
}

int fovi::few_block32(const float* x, int64_t xs, const float* wg, int64_t gs, const float* wu, int64_t us, const float* wd, int64_t ds, int m, int c, int f, int o, const float* bg,
                      const float* bu, const float* bd, int act, float* h, int64_t h_pitch, float* y, cudaStream_t st) {
  auto vec = [](const float* p, int64_t pitch) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && pitch % 4 == 0; };
  const int tokens = (m + 7) / 8;
  const Few32Args up{x, wg, wu, xs, gs, us, m, f, c, act, bg, bu, h, h_pitch, vec(x, xs), vec(wg, gs) && vec(wu, us)};
  FOVI_CUDA(fovi::launch_pdl(product_few32_kernel<true>, dim3((f + ROWS - 1) / ROWS, tokens), 256, 0, st, up));
  int rc = fovi::after_launch("product_few32_kernel");
  if (rc) return rc;
  const Few32Args down{h, wd, nullptr, h_pitch, ds, 0, m, o, f, act, bd, nullptr, y, o, vec(h, h_pitch), vec(wd, ds)};
  FOVI_CUDA(fovi::launch_pdl(product_few32_kernel<false>, dim3((o + ROWS - 1) / ROWS, tokens), 256, 0, st, down));
  return fovi::after_launch("product_few32_kernel");
}

int fovi::few_int8(const FewRows& q, const FewRows& w, int m, int n, int k, const float* scale, const float* wscale, const float* bias, void* y, int y_dtype, cudaStream_t st) {
  FewArgs a = args(q, w, m, n, k, 1);
  a.scale = scale; a.wscale = wscale; a.bias_f = bias; a.y_f32 = y_dtype == FOVI_F32;
  a.y = y; a.y_pitch = n;
  return by_tokens<SCALED>(a, false, st);
}
