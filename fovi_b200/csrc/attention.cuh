// Cross attention: launch arguments shared by its kernels.
#pragma once
#include <limits.h>
#include <math.h>

#include "common.cuh"

namespace fovi {

constexpr int ATT_MAX_DIM = 128;

// q [B, Lq, H, D] over k, v [B, Lk, Hkv, D] (element strides of batch, token and head; channels contiguous); head h reads state head h / (H / Hkv).
struct AttnArgs {
  const void *q, *k, *v, *o, *dy;
  void *out, *dq, *dk, *dv;
  float *lse, *delta;                       // [B, H, Lq]: base-2 logarithm of the row's sum (+inf for a row without a key); rowsum(dy * o)
  const int32_t* lengths;                   // [B] or null: keys at and behind lengths[b] are masked
  const uint8_t* mask;                      // [B, Lk] or null: keys whose byte is 0 are masked
  int64_t q_sb, q_sl, q_sh, k_sb, k_sl, k_sh, v_sb, v_sl, v_sh, g_sb, g_sl, g_sh;
  int B, Lq, Lk, H, Hkv, D, group, vec;     // vec: rows of whole 16-byte pieces on 16-byte boundaries
  int splits;                               // parts of a row's keys, each to part_o [splits][B, Lq, H, D] and (forward) part_lse [splits][B, Lq, H]
  float *part_o, *part_lse;
  float scale, scale_log2;                  // scale_log2 = scale * log2(e): the softmax is taken in base 2
};

// Keys of sample b that lie in front of its length.
__device__ __forceinline__ int key_end(const AttnArgs& a, int b) { return a.lengths ? min(max(__ldg(a.lengths + b), 0), a.Lk) : a.Lk; }

}  // namespace fovi
