// Matrix products of a token block: what their kernels and entry points share.
#pragma once
#include <cuda_bf16.h>

#include "common.cuh"

namespace fovi {

enum { ACT_SILU = 0, ACT_GELU = 1 };

// What a bf16 gated projection writes: h = act(g) u and, for the backward pass, g and u rounded to the upper 24 of their 32 bits, 16 in one tensor and 8 in another: as bf16 their rounding would be
// a third one in every gradient (0.0034 off in place of 0.0023, of which 0.0017 is a result's own rounding).
struct Hidden {
  void* h;                       // [tokens, pitch]
  uint16_t* high; uint8_t* low;  // [tokens, pitch / 32, 2, 32]: g and u of 32 columns side by side, so that a row's piece is 128 and 64 bytes; null where no gradient is wanted
  int64_t pitch;                 // a multiple of 32
};

}  // namespace fovi
