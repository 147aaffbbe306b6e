// Rotary positions with several axes.  x [B, L, H, D]; pair p of a head belongs to one axis a(p) and turns by the angle  t = position[b, l, a(p)] * frequency[p]:
//   (u, v) -> (u cos t - v sin t, v cos t + u sin t)
// `pairing` says which channels a pair is: (p, p + P) of the first 2P ("halves") or (2p, 2p + 1) ("pairs"); channels from 2P on, and the first `prefix` tokens
// (class and register tokens, which have no place), pass as they are.  The gradient is the same map with -t: a rotation's transpose.
// A token's angles are the same for all its heads.  The angle is the exact product, in two float32 parts: cos and sin are taken at the rounded product (whose
// error grows with it: 4e-6 at t = 64) and turned by its rounding error e: cos(t + e) = cos t - e sin t, sin(t + e) = sin t + e cos t, up to e^2.
#include <cuda_bf16.h>
#include <limits.h>

#include "common.cuh"

namespace {

constexpr int MAX_AXES = 4;

struct RotArgs {
  int64_t tokens;                        // B * L
  int L, H, D, P, prefix, axes, ends[MAX_AXES], interleaved, inverse;
  int64_t sb, sl, sh, pos_batch;         // element strides of x; of a sample's positions (0: shared)
  const float *pos, *freq;
};

__device__ __forceinline__ void turn_of(const RotArgs& a, int64_t b, int l, int p, float& c, float& s) {
  int ax = 0;
#pragma unroll
  for (int i = 0; i < MAX_AXES - 1; ++i) ax += i < a.axes - 1 && p >= a.ends[i];
  const float q = __ldg(a.pos + b * a.pos_batch + (int64_t)(l - a.prefix) * a.axes + ax), f = __ldg(a.freq + p);
  const float t = __fmul_rn(q, f), e = __fmaf_rn(q, f, -t);
  float s0, c0;
  sincosf(t, &s0, &c0);
  c = fmaf(-s0, e, c0);
  s = fmaf(c0, e, s0);
  if (a.inverse) s = -s;
}

// One thread per (token, pair) and per channel that passes, all heads.
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
  turn_of(a, b, l, p, c, s);
  for (int h = 0; h < a.H; ++h) {
    const float u = ld_as_float(xt + h * a.sh + c0), v = ld_as_float(xt + h * a.sh + c1);
    yt[h * a.D + c0] = from_float<T>(u * c - v * s);
    yt[h * a.D + c1] = from_float<T>(v * c + u * s);
  }
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
  const int64_t blocks = (a.tokens * (D - P) + 255) / 256;
  if (blocks > INT_MAX) return FOVI_ERR_UNSUPPORTED;
  auto st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == FOVI_BF16) rotary_kernel<__nv_bfloat16><<<(int)blocks, 256, 0, st>>>((const __nv_bfloat16*)x, (__nv_bfloat16*)y, a);
  else rotary_kernel<float><<<(int)blocks, 256, 0, st>>>((const float*)x, (float*)y, a);
  return fovi::after_launch("rotary_kernel");
}
