// Tensor-core cross attention: what the forward and the backward kernels share.  Everything on the device side has internal linkage.
#pragma once
#include "attention.cuh"
#include "pairs.cuh"
#include "tc_common.cuh"

namespace fovi {
// A row's q, k, v ... as the tensor copies see them: an axis that the caller expanded (stride 0) has extent 1 and coordinate 0.
struct TcView { int mul_h, mul_b; };
struct AttnTcArgs {
  AttnArgs a;
  TcView q, k, v, g;
  int splits;              // forward: parts of a row tile's keys, and what each found
  float *part_o, *part_lse;
  int* status;             // wait site at which a kernel gave up
  uint32_t wait_limit;
  int skip_loads;          // self-test: the loads are withheld, so the first wait must give up
};

bool attention_tc_takes(const AttnArgs& a, int dtype, bool backward);
int64_t attention_tc_forward_bytes(int B, int Lq, int Lk, int H, int D);
int launch_attention_tc_forward(const AttnArgs& a, void* work, cudaStream_t st, bool selftest);      // work null: no splits
int64_t attention_tc_backward_bytes(int B, int Lq, int H);
int launch_attention_tc_backward(const AttnArgs& a, void* work, cudaStream_t st, bool selftest);
int attention_tc_check(cudaStream_t st);
int attention_tc_status(int** word);        // the current device's status word
// Boxes of 64 channels x `rows` tokens of a [B, L, H, D] tensor.
int encode_rows(CUtensorMap* m, TcView* view, const void* p, int64_t sb, int64_t sl, int64_t sh, int B, int L, int H, int D, int rows);
}  // namespace fovi

namespace {

constexpr int AT_M = 128;                 // rows of a tile: the M of an MMA, one tensor-memory lane each

// One 64-channel box of a tile: `rows` rows of 128 bytes, 128-byte swizzle.
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
               ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3) : "memory");
}

// The other way; what lies outside the tensor is left out.
__device__ __forceinline__ void tma_store_4d(const CUtensorMap* map, uint32_t src, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4, %5}], [%1];"
               ::"l"(map), "r"(src), "r"(c0), "r"(c1), "r"(c2), "r"(c3) : "memory");
}
// Ends the group of this thread's stores and waits until they have read shared memory.
__device__ __forceinline__ void bulk_commit_and_read() {
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
  asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}

// A from tensor memory (bf16, two per column), B from shared memory.
__device__ __forceinline__ void tc_mma_bf16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
      ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}

__device__ __forceinline__ void tc_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
        "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
               ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
                 "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tc_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Behind tc_ld_wait: what reads the loaded registers stays behind the wait, which does not name them.
template <int N> __device__ __forceinline__ void tc_loaded(uint32_t* r) {
#pragma unroll
  for (int i = 0; i < N; i += 8)
    asm volatile("" : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7]));
}
// Values written to shared memory by threads, seen by the MMAs.
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}

// Instruction descriptor: float32 accumulators, bf16 operands, A K-major, M = 128.
__device__ __forceinline__ constexpr uint32_t at_idesc(int n, bool b_mn_major) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(AT_M >> 4) << 24);
}

// Bounded wait of a converged warp (see mbar_wait).  All lanes ask and leave together: a barrier that is done costs about 90 clocks, where lanes that leave a loop one by one cost 240,
// and these kernels pass four to six such barriers a tile.
__device__ __forceinline__ bool at_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status, int code, uint32_t limit) {
  for (uint32_t it = 0; it < limit; ++it) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    if ((it & 255u) == 255u && __any_sync(0xffffffffu, *abort_flag)) return false;
  }
  *abort_flag = 1;
  atomicCAS(status, 0, code);
  return false;
}

// The products, issued by one lane of a warp that is together.  Operands' descriptors are made by the whole warp and the loops have a fixed number of turns, so that they stay in uniform
// registers, where the instruction takes them from: from a loop of one thread an MMA of N = 64 took 75 clocks to issue instead of 32 to 48.
// D[128, N] = A[128 rows, channels] B[N rows, channels]^T: both tiles K-major, in boxes of 64 channels that are a_box, b_box bytes apart; then `done` is told.
template <int DC> __device__ __forceinline__ void mma_rows(uint32_t d, uint32_t a_smem, uint32_t a_box, uint32_t b_smem, uint32_t b_box, uint32_t idesc) {
  const uint64_t desc = smem_desc(0, 16u, 1024u, 2u), da = desc + (a_smem >> 4), db = desc + (b_smem >> 4);
  if (elect_one()) {
#pragma unroll
    for (int k = 0; k < 4 * DC; ++k)
      tc_mma_bf16(d, da + (k >> 2) * (a_box >> 4) + (k & 3) * 2, db + (k >> 2) * (b_box >> 4) + (k & 3) * 2, idesc, k ? 1u : 0u);
  }
  __syncwarp();
}
// D[128, channels] (+)= A[128, 64 rows] B[64 rows, channels]: A in tensor memory, B the same kind of tile read MN-major; of its four slices of 16 rows the first `steps`.
__device__ __forceinline__ void mma_mix(uint32_t d, uint32_t a_tmem, uint32_t b_smem, uint32_t b_box, int steps, uint32_t idesc, bool accumulate) {
  const uint64_t desc = smem_desc(0, b_box, 1024u, 2u) + (b_smem >> 4);
  if (elect_one()) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < steps) tc_mma_bf16_ts(d, a_tmem + k * 8, desc + k * 128, idesc, accumulate || k ? 1u : 0u);
  }
  __syncwarp();
}

// Bits of the 32 keys from `key`: which may be read.  `all` when there is no mask: only the sample's end counts.
__device__ __forceinline__ uint32_t key_bits(const fovi::AttnArgs& a, const uint8_t* mask, int key, int end, int lane) {
  const int n = end - key;
  uint32_t w = n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
  if (mask) w &= __ballot_sync(0xffffffffu, lane < n && __ldg(mask + key + lane));
  return w;
}

}  // namespace
