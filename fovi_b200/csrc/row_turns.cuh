// Row tiles of the attention gradients' persistent blocks take turns on two operand buffers.  Plain C++ (the host test steps it against a model of the barriers).
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define FOVI_TURN_FN __host__ __device__ __forceinline__
#else
#define FOVI_TURN_FN inline
#endif

namespace fovi {

// Row tile 0, 1, 2, ... of a block is in buffer 0, 1, 0, ...  Its three barriers are the buffer's own: loaded, staged (the results stand in it), empty (they have been copied out).  A wait by
// parity tells a phase from the next one only while the other side cannot complete both before the waiter looks.  Phase n + 1 of a buffer's barriers follows on its refill, which waits for
// "empty" of phase n, and that for "staged" of phase n to have been seen: so none is ever a phase ahead.  One "staged" for both buffers is not like that: nothing in tile i + 1 waits for
// the copies out of tile i, so two of its phases could complete while the copying warp was still busy, which then looked like none.
struct RowTurn {
  uint32_t seq = 0;
  FOVI_TURN_FN uint32_t buffer() const { return seq & 1u; }
  FOVI_TURN_FN uint32_t parity() const { return seq >> 1 & 1u; }
  FOVI_TURN_FN void next() { ++seq; }
};

}  // namespace fovi
