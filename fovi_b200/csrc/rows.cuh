// Rows held in registers by teams of threads: what the norms over the last axis share.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "common.cuh"
#include "pairs.cuh"

namespace {

template <typename T, int VEC> struct Piece { uint32_t w[sizeof(T) * VEC / 4]; };
template <> struct Piece<__nv_bfloat16, 1> { unsigned short w[1]; };

template <typename T, int VEC> __device__ __forceinline__ Piece<T, VEC> load_piece(const T* p) {
  Piece<T, VEC> r;
  constexpr int B = sizeof(T) * VEC;
  if constexpr (B == 16) *reinterpret_cast<uint4*>(&r) = __ldg(reinterpret_cast<const uint4*>(p));
  else if constexpr (B == 8) *reinterpret_cast<uint2*>(&r) = __ldg(reinterpret_cast<const uint2*>(p));
  else if constexpr (B == 4) r.w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
  else r.w[0] = __ldg(reinterpret_cast<const unsigned short*>(p));
  return r;
}
template <typename T, int VEC> __device__ __forceinline__ void widen(const Piece<T, VEC>& r, float* v) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = __uint_as_float(r.w[i]);
  } else if constexpr (VEC == 1) {
    v[0] = __uint_as_float((uint32_t)r.w[0] << 16);
  } else {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) { v[2 * i] = __uint_as_float(r.w[i] << 16); v[2 * i + 1] = __uint_as_float(r.w[i] & 0xffff0000u); }
  }
}
template <typename T, int VEC> __device__ __forceinline__ void store_piece(T* p, const float* v) {
  constexpr int B = sizeof(T) * VEC;
  if constexpr (sizeof(T) == 4) {
    if constexpr (VEC == 4) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    else p[0] = v[0];
  } else if constexpr (VEC == 1) {
    p[0] = __float2bfloat16_rn(v[0]);
  } else {
    uint32_t w[VEC / 2];
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    if constexpr (B == 16) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Where a thread's pieces lie, and which rows its team takes.
template <int VEC, bool BLOCK> struct Team {
  int first, pitch, warp, warps;
  int64_t row, step;
  __device__ __forceinline__ Team() {
    warp = threadIdx.x >> 5; warps = blockDim.x >> 5;
    const int lane = BLOCK ? threadIdx.x : threadIdx.x & 31;
    first = lane * VEC;
    pitch = (BLOCK ? blockDim.x : 32) * VEC;
    row = BLOCK ? blockIdx.x : (int64_t)blockIdx.x * warps + warp;
    step = BLOCK ? gridDim.x : (int64_t)gridDim.x * warps;
  }
};

// Threads of the largest block: single values take more instructions and more registers.
template <int VEC> constexpr int BLOCK_MOST = VEC == 1 ? 512 : 1024;

// As many blocks as the SMs hold at once: every team then takes the same number of rows.  `known`: the answer for one SM, which threads that ask at once all store.
template <typename Kernel> int64_t resident(Kernel k, int threads, size_t smem, std::atomic<int>& known) {
  int n = known.load(std::memory_order_relaxed);
  if (!n) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, k, threads, smem) != cudaSuccess || n < 1) n = 1;
    known.store(n, std::memory_order_relaxed);
  }
  return (int64_t)fovi::sm_count() * n;
}

// Values two by two, for the instructions that take two.
template <int E> struct Pairs {
  static_assert(E % 2 == 0, "an even number of values a thread");
  float2 v[E / 2];
  __device__ __forceinline__ float* at(int i) { return reinterpret_cast<float*>(v) + i; }
};

}  // namespace
