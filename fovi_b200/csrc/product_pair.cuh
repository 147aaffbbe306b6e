// Building blocks of the products on CTA pairs (product_tc.cu, product_split.cu).
#pragma once
#include <cuda_bf16.h>

#include <atomic>

#include "pairs.cuh"
#include "tc_common.cuh"

namespace {

__device__ __forceinline__ uint32_t pt_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t pt_map(uint32_t local, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(local), "r"(rank));
  return r;
}
__device__ __forceinline__ void pt_sync() { asm volatile("barrier.cluster.arrive.release;\n barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ void pt_load(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
               ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1) : "memory");
}
template <bool I8> __device__ __forceinline__ void pt_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if (I8)
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}\n"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
  else
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void pt_commit(uint32_t bar) {            // on the barrier at this offset in both CTAs
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
}
// Behind tc_ld_wait: what reads the loaded registers stays behind the wait, which does not name them.
__device__ __forceinline__ void pt_loaded(uint32_t (&r)[32]) {
#pragma unroll
  for (int i = 0; i < 32; i += 8)
    asm volatile("" : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7]));
}
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
__device__ __forceinline__ void st_global_32f(float* p, const uint32_t* v) {
  const uint32_t w[8] = {v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]};
  st_global_32(p, w);
}

// What a launch asks the runtime once for each device (of the first 64; of others every time): a kernel's shared memory, a status word's address.
inline int device_slot() {
  int dev = -1;
  return cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64 ? dev : -1;
}
template <typename Kernel> cudaError_t allow_shared(Kernel kernel, int bytes, std::atomic<uint64_t>& done) {
  const int dev = device_slot();
  if (dev >= 0 && (done.load(std::memory_order_relaxed) >> dev & 1)) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev >= 0) done.fetch_or(1ull << dev, std::memory_order_relaxed);
  return e;
}
template <typename Symbol> cudaError_t word_of(int** word, Symbol& symbol, std::atomic<int*> (&known)[64]) {
  const int dev = device_slot();
  if (dev >= 0 && (*word = known[dev].load(std::memory_order_relaxed))) return cudaSuccess;
  const cudaError_t e = cudaGetSymbolAddress(reinterpret_cast<void**>(word), symbol);
  if (e == cudaSuccess && dev >= 0) known[dev].store(*word, std::memory_order_relaxed);
  return e;
}

}  // namespace
