// Matrix products of a token block: what their kernels and entry points share.
#pragma once
#include <cuda_bf16.h>

#include "common.cuh"

namespace fovi {

// Element (i, k) of an operand is p[i * row + k * step]: one of the two strides is 1.
struct Operand { const void* p; int64_t row, step; };

enum { ACT_SILU = 0, ACT_GELU = 1 };

// What a gated projection writes: act(g) u and, for the backward pass, g and u.  Of bf16 blocks g and u are kept as the upper 24 of their 32 bits, 16 in one tensor and 8 in another:
// as bf16 their rounding would be a third one in every gradient (0.0034 off in place of 0.0023, of which 0.0017 is a result's own rounding).
struct Hidden {
  void* h;                       // [tokens, pitch] of the block's type
  float *g, *u;                  // [tokens, pitch], float32 blocks; these and the next two are null where no gradient is wanted
  uint16_t* high; uint8_t* low;  // [tokens, pitch / 32, 2, 32], bf16 blocks: g and u of 32 columns side by side, so that a row's piece is 128 and 64 bytes
  int64_t pitch;                 // a multiple of 32
};

}  // namespace fovi
