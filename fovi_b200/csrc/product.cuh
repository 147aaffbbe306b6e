// Matrix products of a token block: what their kernels and entry points share.
#pragma once
#include <cuda_bf16.h>

#include "common.cuh"

namespace fovi {

// Element (i, k) of an operand is p[i * row + k * step]: one of the two strides is 1.
struct Operand { const void* p; int64_t row, step; };

enum { ACT_SILU = 0, ACT_GELU = 1 };

// What a gated projection writes: act(g) u and, for the backward pass, g and u.  Of bf16 blocks g and u are kept as the upper 24 of their 32 bits, 16 in one tensor and 8 in another:
// as bf16 their rounding would be a third one in every gradient (0.0034 off in place of 0.0024, of which 0.0017 is a result's own rounding).
struct Hidden {
  void *h, *g, *u;               // [tokens, pitch] of the block's type; g and u null where no gradient is wanted
  uint8_t *g_low, *u_low;        // [tokens, pitch], bf16 blocks
  int64_t pitch;
};

}  // namespace fovi

namespace {

__device__ __forceinline__ float upper24(uint32_t high, uint32_t low) { return __uint_as_float(high << 16 | low << 8 | 0x80u); }

}  // namespace
