// Gated feed-forward block on tokens x [tokens, C]:
//   g = x Wg^T + bg,  u = x Wu^T + bu,  h = act(g) u,  y = h Wd^T + bd          Wg, Wu [F, C], Wd [O, F]; act(g) = g s(g) (s: logistic) or g Phi(g) (Phi: normal distribution)
// and its gradients
//   dh = dy Wd,  dg = dh u act'(g),  du = dh act(g),  dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x,  dWd = dy^T h,  and column sums of dg, du, dy for the biases.
#include <algorithm>

#include "product.cuh"
#include "product_simt.cuh"

using fovi::Hidden;
using fovi::Operand;

namespace {

template <typename T> __device__ __forceinline__ float bias_at(const void* b, int n) { return b ? ld_as_float(static_cast<const T*>(b) + n) : 0.f; }

// act(g) and act'(g)
__device__ __forceinline__ float2 activate(float g, int act) {
  if (act == fovi::ACT_SILU) {
    const float p = 1.f / (1.f + expf(-g)), a = g * p;
    return make_float2(a, fmaf(a, 1.f - p, p));
  }
  const float p = 0.5f * (1.f + erff(g * 0.70710678118654752f));
  return make_float2(g * p, fmaf(g * 0.39894228040143268f, expf(-0.5f * g * g), p));
}

template <typename T> struct GateUp {       // g and u -> h
  Hidden to; const void *bg, *bu; int act;
  __device__ __forceinline__ void operator()(int64_t m, int n, float g, float u) const {
    g += bias_at<T>(bg, n);
    u += bias_at<T>(bu, n);
    const int64_t at = m * to.pitch + n;
    if (to.g) {
      if (sizeof(T) == 4) {
        static_cast<float*>(to.g)[at] = g;
        static_cast<float*>(to.u)[at] = u;
      } else {
        const uint32_t gb = __float_as_uint(g), ub = __float_as_uint(u);
        static_cast<uint16_t*>(to.g)[at] = gb >> 16;
        static_cast<uint16_t*>(to.u)[at] = ub >> 16;
        to.g_low[at] = gb >> 8;
        to.u_low[at] = ub >> 8;
      }
    }
    static_cast<T*>(to.h)[at] = from_float<T>(activate(g, act).x * u);
  }
};
template <typename T> struct HiddenGrad {   // dh -> dg, du
  Hidden from; T *dg, *du; int act;
  __device__ __forceinline__ void operator()(int64_t m, int n, float dh, float) const {
    const int64_t at = m * from.pitch + n;
    float g, u;
    if (sizeof(T) == 4) {
      g = static_cast<const float*>(from.g)[at];
      u = static_cast<const float*>(from.u)[at];
    } else {
      g = upper24(static_cast<const uint16_t*>(from.g)[at], from.g_low[at]);
      u = upper24(static_cast<const uint16_t*>(from.u)[at], from.u_low[at]);
    }
    const float2 s = activate(g, act);
    dg[at] = from_float<T>(dh * u * s.y);
    du[at] = from_float<T>(dh * s.x);
  }
};
template <typename T> struct Store {
  T* y; int64_t pitch; const void* bias;
  __device__ __forceinline__ void operator()(int64_t m, int n, float v, float) const { y[m * pitch + n] = from_float<T>(v + bias_at<T>(bias, n)); }
};

// Column sums of [rows, n] in a fixed order: parts of 64 rows' strips, then their sum.
template <typename T>
__global__ void __launch_bounds__(128) column_parts_kernel(const T* x, int64_t rows, int n, int64_t pitch, int strips, float* part) {
  const int c = blockIdx.x * 128 + threadIdx.x;
  if (c >= n) return;
  float s = 0.f;
  for (int64_t r = blockIdx.y; r < rows; r += strips) s += ld_as_float(x + r * pitch + c);
  part[(size_t)blockIdx.y * n + c] = s;
}
template <typename T>
__global__ void __launch_bounds__(1024) column_join_kernel(const float* part, int parts, int n, T* out) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < n)
    for (int p = w; p < parts; p += 32) s += part[(size_t)p * n + c];
  red[w][lane] = s;
  __syncthreads();
  if (w || c >= n) return;
  s = 0.f;
  for (int i = 0; i < 32; ++i) s += red[i][lane];
  out[c] = from_float<T>(s);
}
constexpr int STRIPS = 64;
template <typename T> int column_sums(const void* x, int64_t rows, int n, int64_t pitch, float* part, void* out, cudaStream_t st) {
  const int strips = (int)std::min<int64_t>(STRIPS, rows);
  column_parts_kernel<T><<<dim3((n + 127) / 128, strips), 128, 0, st>>>(static_cast<const T*>(x), rows, n, pitch, strips, part);
  const int rc = fovi::after_launch("column_parts_kernel");
  if (rc) return rc;
  column_join_kernel<T><<<(n + 31) / 32, 1024, 0, st>>>(part, strips, n, static_cast<T*>(out));
  return fovi::after_launch("column_join_kernel");
}

int64_t pitch_of(int F) { return ((int64_t)F + 31) / 32 * 32; }
// Where the parts of a buffer for the hidden values lie.
Hidden hidden_at(void* p, int dtype, int64_t M, int F, bool saved) {
  Hidden h{};
  h.pitch = pitch_of(F);
  const int64_t n = M * h.pitch, size = fovi::dtype_size(dtype);
  char* at = static_cast<char*>(p);
  h.h = at;
  if (saved) {
    h.g = at + n * size;
    h.u = at + 2 * n * size;
    h.g_low = reinterpret_cast<uint8_t*>(at + 3 * n * size);
    h.u_low = h.g_low + n;
  }
  return h;
}

struct Block {
  const void *x, *wg, *wu, *wd, *bg, *bu, *bd;
  int64_t M, xs, gs, us, ds; int C, F, O, act;
};

template <typename T> int forward(const Block& b, void* y, const Hidden& hid, cudaStream_t st) {
  SimtArgs p{};
  p.m = b.M; p.n = b.F; p.k[0] = b.C; p.segments = 1;
  p.a[0] = Operand{b.x, b.xs, 1};
  p.b[0] = Operand{b.wg, b.gs, 1};
  p.b2 = Operand{b.wu, b.us, 1};
  int rc = product_simt<T, true>(p, GateUp<T>{hid, b.bg, b.bu, b.act}, st);
  if (rc) return rc;
  p.n = b.O; p.k[0] = b.F;
  p.a[0] = Operand{hid.h, hid.pitch, 1};
  p.b[0] = Operand{b.wd, b.ds, 1};
  return product_simt<T, false>(p, Store<T>{static_cast<T*>(y), b.O, b.bd}, st);
}

struct Grads { const void* dy; int64_t dys; void *dx, *dwg, *dwu, *dwd, *dbg, *dbu, *dbd; };

template <typename T> int backward(const Block& b, const Hidden& hid, const Grads& g, char* work, cudaStream_t st) {
  T *dg = reinterpret_cast<T*>(work), *du = dg + b.M * hid.pitch;
  float* part = reinterpret_cast<float*>(du + b.M * hid.pitch);
  int rc;
  SimtArgs p{};
  p.segments = 1;
  if (g.dx || g.dwg || g.dwu || g.dbg || g.dbu) {
    p.m = b.M; p.n = b.F; p.k[0] = b.O;
    p.a[0] = Operand{g.dy, g.dys, 1};
    p.b[0] = Operand{b.wd, 1, b.ds};
    if ((rc = product_simt<T, false>(p, HiddenGrad<T>{hid, dg, du, b.act}, st))) return rc;
  }
  if (g.dx) {
    p.m = b.M; p.n = b.C; p.k[0] = p.k[1] = b.F; p.segments = 2;
    p.a[0] = Operand{dg, hid.pitch, 1}; p.a[1] = Operand{du, hid.pitch, 1};
    p.b[0] = Operand{b.wg, 1, b.gs}; p.b[1] = Operand{b.wu, 1, b.us};
    if ((rc = product_simt<T, false>(p, Store<T>{static_cast<T*>(g.dx), b.C, nullptr}, st))) return rc;
  }
  p.segments = 1;
  p.k[0] = (int)b.M;
  const struct { void* to; const void* a; int64_t as; int m; const void* b; int64_t bs; int n; } weights[3] = {
      {g.dwg, dg, hid.pitch, b.F, b.x, b.xs, b.C}, {g.dwu, du, hid.pitch, b.F, b.x, b.xs, b.C}, {g.dwd, g.dy, g.dys, b.O, hid.h, hid.pitch, b.F}};
  for (const auto& w : weights) {
    if (!w.to) continue;
    p.m = w.m; p.n = w.n;
    p.a[0] = Operand{w.a, 1, w.as};
    p.b[0] = Operand{w.b, 1, w.bs};
    if ((rc = product_simt<T, false>(p, Store<T>{static_cast<T*>(w.to), w.n, nullptr}, st))) return rc;
  }
  if (g.dbg && (rc = column_sums<T>(dg, b.M, b.F, hid.pitch, part, g.dbg, st))) return rc;
  if (g.dbu && (rc = column_sums<T>(du, b.M, b.F, hid.pitch, part, g.dbu, st))) return rc;
  if (g.dbd && (rc = column_sums<T>(g.dy, b.M, b.O, g.dys, part, g.dbd, st))) return rc;
  return FOVI_OK;
}

bool valid(int dtype, int64_t M, int C, int F, int O) { return fovi::valid_dtype(dtype) && M >= 0 && M <= (1 << 30) && C >= 1 && F >= 1 && O >= 1; }

}  // namespace

extern "C" int64_t fovi_gated_ffn_saved_bytes(int dtype, int64_t tokens, int F) {
  if (!valid(dtype, tokens, 1, F, 1)) return -1;
  return tokens * pitch_of(F) * (dtype == FOVI_BF16 ? 8 : 12);
}

extern "C" int64_t fovi_gated_ffn_workspace_bytes(int dtype, int64_t tokens, int C, int F, int O, int backward) {
  if (!valid(dtype, tokens, C, F, O)) return -1;
  const int64_t n = tokens * pitch_of(F) * (int64_t)fovi::dtype_size(dtype);
  return backward ? 2 * n + (int64_t)STRIPS * std::max(F, O) * 4 : n;
}

extern "C" int fovi_gated_ffn_forward(const void* x, int dtype, int64_t tokens, int C, int F, int O, int64_t x_stride, const void* gate_weight, int64_t gate_stride,
                                      const void* up_weight, int64_t up_stride, const void* down_weight, int64_t down_stride, const void* gate_bias, const void* up_bias,
                                      const void* down_bias, int activation, void* y, void* saved, void* work, int64_t work_bytes, void* stream) {
  if (!valid(dtype, tokens, C, F, O) || activation < 0 || activation > 1 || x_stride < 0 || gate_stride < 0 || up_stride < 0 || down_stride < 0) return FOVI_ERR_INVALID_ARGUMENT;
  if (tokens == 0) return FOVI_OK;
  if (!x || !gate_weight || !up_weight || !down_weight || !y) return FOVI_ERR_INVALID_ARGUMENT;
  if (!saved && (!work || work_bytes < fovi_gated_ffn_workspace_bytes(dtype, tokens, C, F, O, 0))) return FOVI_ERR_INVALID_ARGUMENT;
  const Block b{x, gate_weight, up_weight, down_weight, gate_bias, up_bias, down_bias, tokens, x_stride, gate_stride, up_stride, down_stride, C, F, O, activation};
  const Hidden h = hidden_at(saved ? saved : work, dtype, tokens, F, saved != nullptr);
  auto st = reinterpret_cast<cudaStream_t>(stream);
  return dtype == FOVI_BF16 ? forward<__nv_bfloat16>(b, y, h, st) : forward<float>(b, y, h, st);
}

extern "C" int fovi_gated_ffn_backward(const void* x, int dtype, int64_t tokens, int C, int F, int O, int64_t x_stride, const void* gate_weight, int64_t gate_stride,
                                       const void* up_weight, int64_t up_stride, const void* down_weight, int64_t down_stride, int activation, const void* saved,
                                       const void* dy, int64_t dy_stride, void* dx, void* dgate_weight, void* dup_weight, void* ddown_weight, void* dgate_bias,
                                       void* dup_bias, void* ddown_bias, void* work, int64_t work_bytes, void* stream) {
  if (!valid(dtype, tokens, C, F, O) || activation < 0 || activation > 1 || x_stride < 0 || gate_stride < 0 || up_stride < 0 || down_stride < 0 || dy_stride < 0)
    return FOVI_ERR_INVALID_ARGUMENT;
  auto st = reinterpret_cast<cudaStream_t>(stream);
  const size_t size = fovi::dtype_size(dtype);
  if (tokens == 0) {
    const struct { void* p; size_t n; } zero[] = {{dgate_weight, (size_t)F * C}, {dup_weight, (size_t)F * C}, {ddown_weight, (size_t)O * F},
                                                  {dgate_bias, (size_t)F}, {dup_bias, (size_t)F}, {ddown_bias, (size_t)O}};
    for (const auto& z : zero)
      if (z.p) FOVI_CUDA(cudaMemsetAsync(z.p, 0, z.n * size, st));
    return FOVI_OK;
  }
  if (!x || !gate_weight || !up_weight || !down_weight || !saved || !dy || !work || work_bytes < fovi_gated_ffn_workspace_bytes(dtype, tokens, C, F, O, 1))
    return FOVI_ERR_INVALID_ARGUMENT;
  const Block b{x, gate_weight, up_weight, down_weight, nullptr, nullptr, nullptr, tokens, x_stride, gate_stride, up_stride, down_stride, C, F, O, activation};
  const Hidden h = hidden_at(const_cast<void*>(saved), dtype, tokens, F, true);
  const Grads g{dy, dy_stride, dx, dgate_weight, dup_weight, ddown_weight, dgate_bias, dup_bias, ddown_bias};
  return dtype == FOVI_BF16 ? backward<__nv_bfloat16>(b, h, g, static_cast<char*>(work), st) : backward<float>(b, h, g, static_cast<char*>(work), st);
}
