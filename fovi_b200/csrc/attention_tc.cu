// Cross attention on the tensor cores: bf16 q, k, v of up to 128 channels a head (a multiple of 8), 16-byte aligned rows.
//
// Forward.  One CTA per (128 queries, head, sample), two CTAs per SM; keys in tiles of 64.  Per tile
//   S = Q K^T     SS MMA, M = 128, N = 64, into one of two places in tensor memory
//   P = 2^(scale log2(e) (S - m))     four warps, a thread per query: its row of S in registers, its maximum and sum in two more; P goes back over S as bf16
//   O += P V      TS MMA: P from tensor memory, the tile of V read MN-major, so nothing is transposed
// A TMA warp keeps the rings of K and V tiles full, an MMA warp issues both products.  While the exponentials of one tile are computed the scores of the next are; the other CTA of
// the SM fills what gaps remain.  The reference value m of a row only moves when its maximum has risen
// by more than 8 (in base 2): P then stays below 2^8, bf16's relative rounding is the same at any size, and the pass over O that a move costs is rare.
// Tensor memory (256 columns): S and P [0, 64) and [64, 128), O behind.
// Masked keys: their scores are -inf by a select and their rows of V are set to zero in shared memory, so what they hold has no effect.  A warp whose
// 32 queries lie behind the last one skips the arithmetic.
#include <cuda_bf16.h>

#include "attention_tc.cuh"

using fovi::AttnArgs;
using fovi::AttnTcArgs;
using fovi::key_end;

namespace {

__device__ int g_status;           // wait site at which a kernel gave up, see fovi_attention_check: one word per device
constexpr int AT_THREADS = 192;
constexpr float AT_INF = __builtin_huge_valf();

constexpr int KT = 64;             // keys of a tile

template <int DC> struct Fwd {                     // DC: 64-channel boxes of a row
  static constexpr int NK = DC == 1 ? 4 : 2, NV = NK;
  static constexpr uint32_t BOX = KT * 128u, TILE = DC * BOX, QBOX = AT_M * 128u, QTILE = DC * QBOX;
  static constexpr uint32_t SMEM = 1024 + 1024 + QTILE + (NK + NV) * TILE;
  static constexpr uint32_t O_COL = 2 * KT;
};

struct FwdHeader {
  uint64_t q_full, k_full[4], k_empty[4], v_full[4], v_empty[4], s_full[2], p_full, o_full, drain;
  uint32_t tmem_base;
  int abort_flag;
};

template <int DC>
__global__ void __launch_bounds__(AT_THREADS, 2)
attn_tc_forward_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const AttnTcArgs t) {
  using F = Fwd<DC>;
  const AttnArgs& a = t.a;
  extern __shared__ unsigned char smem_raw[];
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  FwdHeader* hdr = reinterpret_cast<FwdHeader*>(smem_raw + (base - raw));
  const uint32_t sq = base + 1024, sk = sq + F::QTILE, sv = sk + F::NK * F::TILE;
  volatile int* abort_flag = &hdr->abort_flag;
  const int warp = warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&hdr->q_full), 1);
    for (int i = 0; i < 4; ++i) {
      mbar_init(smem_u32(&hdr->k_full[i]), 1); mbar_init(smem_u32(&hdr->k_empty[i]), 1);
      mbar_init(smem_u32(&hdr->v_full[i]), 1); mbar_init(smem_u32(&hdr->v_empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) mbar_init(smem_u32(&hdr->s_full[i]), 1);
    mbar_init(smem_u32(&hdr->p_full), 4); mbar_init(smem_u32(&hdr->o_full), 1);
    mbar_init(smem_u32(&hdr->drain), 1);
    hdr->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 4) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&hdr->tmem_base)), "r"(256u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int n_qt = (a.Lq + AT_M - 1) / AT_M;
  const int q0 = (int)(blockIdx.x % n_qt) * AT_M, h = blockIdx.x / n_qt % a.H, b = blockIdx.x / n_qt / a.H, hk = h / a.group;
  const int end = key_end(a, b), tiles = (end + KT - 1) / KT;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = hdr->tmem_base;

  if (warp == 5) {
    // ------------------------------------------------------------ tensor copies
    if (lane == 0 && tiles > 0 && !t.skip_loads) {
      const uint32_t qf = smem_u32(&hdr->q_full);
      mbar_expect_tx(qf, F::QTILE);
      for (int c = 0; c < DC; ++c) tma_load_4d(sq + c * F::QBOX, &tm_q, qf, 64 * c, q0, h * t.q.mul_h, b * t.q.mul_b);
      uint32_t ks = 0, kp = 0, vs = 0, vp = 0;
      for (int j = 0; j < tiles; ++j) {
        if (!mbar_wait(smem_u32(&hdr->k_empty[ks]), kp ^ 1u, abort_flag, t.status, 1, t.wait_limit)) break;
        const uint32_t kf = smem_u32(&hdr->k_full[ks]);
        mbar_expect_tx(kf, F::TILE);
        for (int c = 0; c < DC; ++c) tma_load_4d(sk + ks * F::TILE + c * F::BOX, &tm_k, kf, 64 * c, j * KT, hk * t.k.mul_h, b * t.k.mul_b);
        if (++ks == F::NK) { ks = 0; kp ^= 1u; }
        if (!mbar_wait(smem_u32(&hdr->v_empty[vs]), vp ^ 1u, abort_flag, t.status, 2, t.wait_limit)) break;
        const uint32_t vf = smem_u32(&hdr->v_full[vs]);
        mbar_expect_tx(vf, F::TILE);
        for (int c = 0; c < DC; ++c) tma_load_4d(sv + vs * F::TILE + c * F::BOX, &tm_v, vf, 64 * c, j * KT, hk * t.v.mul_h, b * t.v.mul_b);
        if (++vs == F::NV) { vs = 0; vp ^= 1u; }
      }
      if (*abort_flag)      // copies in flight get time to land before the block leaves its shared memory
        for (int i = 0; i < 64; ++i) __nanosleep(1000);
    }
  } else if (warp == 4) {
    // ------------------------------------------------------------ MMAs (all lanes loop, one issues: see elect_one)
    const int dsteps = (a.D + 15) / 16;
    const uint32_t id_s = at_idesc(KT, false), id_o = at_idesc(dsteps * 16, true);
    const uint32_t u_sq = warp_uniform(sq), u_sk = warp_uniform(sk), u_sv = warp_uniform(sv), u_tmem = warp_uniform(tmem);
    uint32_t ks = 0, kp = 0, vs = 0, vp = 0;
    bool ok = tiles == 0 || mbar_wait_warp(smem_u32(&hdr->q_full), 0, abort_flag, t.status, 3, t.wait_limit);
    auto scores = [&](int j) {
      if (!mbar_wait_warp(smem_u32(&hdr->k_full[ks]), kp, abort_flag, t.status, 4, t.wait_limit)) return false;
      if (j > 1 && !mbar_wait_warp(smem_u32(&hdr->o_full), j & 1, abort_flag, t.status, 5, t.wait_limit)) return false;      // P of tile j - 2, in the same columns, is read
      tc_fence_after();
      if (elect_one()) {
        mma_rows(u_tmem + (j & 1) * KT, u_sq, F::QBOX, u_sk + ks * F::TILE, F::BOX, dsteps, id_s);
        tc_commit(smem_u32(&hdr->k_empty[ks]));
        tc_commit(smem_u32(&hdr->s_full[j & 1]));
      }
      __syncwarp();
      if (++ks == F::NK) { ks = 0; kp ^= 1u; }
      return true;
    };
    if (ok && tiles > 0) ok = scores(0);
    if (ok && tiles > 1) ok = scores(1);
    for (int j = 0; j < tiles && ok; ++j) {
      ok = mbar_wait_warp(smem_u32(&hdr->v_full[vs]), vp, abort_flag, t.status, 6, t.wait_limit);
      ok = ok && mbar_wait_warp(smem_u32(&hdr->p_full), j & 1, abort_flag, t.status, 7, t.wait_limit);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        mma_mix(u_tmem + F::O_COL, u_tmem + (j & 1) * KT, u_sv + vs * F::TILE, F::BOX, KT / 16, id_o, j > 0);
        tc_commit(smem_u32(&hdr->v_empty[vs]));
        tc_commit(smem_u32(&hdr->o_full));
      }
      __syncwarp();
      if (++vs == F::NV) { vs = 0; vp ^= 1u; }
      if (j + 2 < tiles) ok = scores(j + 2);
    }
    if (*abort_flag && elect_one()) {      // no MMA may still be reading shared memory or writing tensor memory
      tc_commit(smem_u32(&hdr->drain));
      for (uint32_t it = 0; it < (1u << 20); ++it)
        if (mbar_try_wait(smem_u32(&hdr->drain), 0)) break;
    }
  } else {
    // ------------------------------------------------------------ softmax: thread = query
    const int row = q0 + threadIdx.x;
    const bool idle = q0 + warp * 32 >= a.Lq;          // no query in this warp
    const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
    const uint8_t* mask = a.mask ? a.mask + (int64_t)b * a.Lk : nullptr;
    const float c = a.scale_log2;
    float m = -AT_INF;                 // the row's reference value, in units of S
    float2 l = make_float2(0.f, 0.f);
    bool ok = true;
    for (int j = 0; j < tiles; ++j) {
      uint32_t bits[KT / 32];
      bool whole = true;
#pragma unroll
      for (int i = 0; i < KT / 32; ++i) { bits[i] = key_bits(a, mask, j * KT + 32 * i, end, lane); whole = whole && bits[i] == 0xffffffffu; }
      ok = mbar_wait_warp(smem_u32(&hdr->s_full[j & 1]), j >> 1 & 1, abort_flag, t.status, 8, t.wait_limit);
      if (!ok) break;
      tc_fence_after();
      bool move = false;
      float f = 1.f;
      if (!idle) {
        const uint32_t at = lanes + (j & 1) * KT;
        float x[KT];
#pragma unroll
        for (int i = 0; i < KT; i += 32) tc_ld32(at + i, reinterpret_cast<uint32_t*>(x) + i);
        tc_ld_wait();
        tc_loaded<KT>(reinterpret_cast<uint32_t*>(x));
        if (!whole) {
#pragma unroll
          for (int i = 0; i < KT; ++i) x[i] = bits[i >> 5] >> (i & 31) & 1u ? x[i] : -AT_INF;
        }
        float top[4] = {m, x[0], x[1], x[2]};
        top[0] = fmaxf(top[0], x[3]);
#pragma unroll
        for (int i = 4; i < KT; i += 4) {
          if (i & 4) { top[0] = max3(top[0], x[i], x[i + 1]); top[1] = max3(top[1], x[i + 2], x[i + 3]); }
          else { top[2] = max3(top[2], x[i], x[i + 1]); top[3] = max3(top[3], x[i + 2], x[i + 3]); }
        }
        const float m_new = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        move = (m_new - m) * c > 8.f;
        if (move) { f = ex2((m - m_new) * c); m = m_new; l = mul2(l, make_float2(f, f)); }
        const float mc = m == -AT_INF ? 0.f : m * c;      // no key yet: every exponent is -inf
#pragma unroll
        for (int i = 0; i < KT; i += 2) {
          const float2 e = fma2(make_float2(x[i], x[i + 1]), make_float2(c, c), make_float2(-mc, -mc));
          const float2 p = make_float2(ex2(e.x), ex2(e.y));
          l = add2(l, p);
          x[i >> 1] = __uint_as_float(pack_bf16(p.x, p.y));
        }
        tc_st32(at, reinterpret_cast<uint32_t*>(x));       // over S, which is in registers
      }
      if (j > 0) {
        // The product with the previous P is done: O is this thread's.  Every warp waits here in every tile: one that ran ahead would meet barriers a phase behind
        // the one that it means, which look the same as those a phase ahead.
        ok = mbar_wait_warp(smem_u32(&hdr->o_full), (j - 1) & 1, abort_flag, t.status, 9, t.wait_limit);
        if (!ok) break;
        if (__any_sync(0xffffffffu, move)) {
          tc_fence_after();
#pragma unroll
          for (int o = 0; o < DC * 64; o += 32) {
            uint32_t r[32];
            tc_ld32(lanes + F::O_COL + o, r);
            tc_ld_wait();
            tc_loaded<32>(r);
#pragma unroll
            for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * f);
            tc_st32(lanes + F::O_COL + o, r);
          }
        }
      }
      if (!whole) {                     // rows of V that must not be read: a zero weight times what they hold need not be zero
        ok = mbar_wait_warp(smem_u32(&hdr->v_full[j % F::NV]), (j / F::NV) & 1, abort_flag, t.status, 10, t.wait_limit);
        if (!ok) break;
        if (threadIdx.x < KT) {
          const int r = threadIdx.x;
          uint32_t word = bits[0];
#pragma unroll
          for (int i = 1; i < KT / 32; ++i) word = (r >> 5) == i ? bits[i] : word;
          if (!(word >> (r & 31) & 1u)) {
            unsigned char* v = smem_raw + (sv - raw) + (j % F::NV) * F::TILE + r * 128;
#pragma unroll
            for (int i = 0; i < DC * 8; ++i) *reinterpret_cast<uint4*>(v + (i >> 3) * F::BOX + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_async_smem();
        }
      }
      tc_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&hdr->p_full));
    }
    if (ok && tiles > 0) ok = mbar_wait_warp(smem_u32(&hdr->o_full), (tiles - 1) & 1, abort_flag, t.status, 11, t.wait_limit);
    if (ok && !idle) {
      tc_fence_after();
      const bool none = m == -AT_INF;
      const float sum = l.x + l.y, inv = none ? 0.f : 1.f / sum;
      // `none` also holds for a row of scores that are all not a number; its sum is not a number then, and so is its result
      const bool zero = none && !(sum != sum);
      __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + (((int64_t)b * a.Lq + row) * a.H + h) * a.D;
#pragma unroll
      for (int o = 0; o < DC * 64; o += 32) {
        uint32_t r[32];
        if (tiles > 0) { tc_ld32(lanes + F::O_COL + o, r); tc_ld_wait(); tc_loaded<32>(r); }
        if (row < a.Lq) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            if (o + 8 * g < a.D) {
              uint32_t w[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float u = __uint_as_float(r[8 * g + 2 * i]) * inv, v = __uint_as_float(r[8 * g + 2 * i + 1]) * inv;
                w[i] = zero ? 0u : pack_bf16(none ? sum : u, none ? sum : v);
              }
              *reinterpret_cast<uint4*>(out + o + 8 * g) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        }
        __syncwarp();
      }
      if (a.lse && row < a.Lq) a.lse[((int64_t)b * a.H + h) * a.Lq + row] = zero ? AT_INF : m * c + log2f(sum);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 4) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256u) : "memory");
}

// ------------------------------------------------------------------------------------------------------------ host
bool rows_ok(const void* p, int64_t sb, int64_t sl, int64_t sh, int B, int L, int H) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (L == 1 || (sl > 0 && sl % 8 == 0)) && (H == 1 || sh % 8 == 0) && (B == 1 || sb % 8 == 0) &&
         sl < (int64_t)1 << 38 && sh < (int64_t)1 << 38 && sb < (int64_t)1 << 38;
}

template <int DC>
int forward(const AttnArgs& a, cudaStream_t st, bool selftest) {
  using F = Fwd<DC>;
  CUtensorMap tq, tk, tv;
  AttnTcArgs t = {};
  t.a = a;
  t.wait_limit = selftest ? 4096u : WAIT_LIMIT;
  t.skip_loads = selftest;
  int rc = fovi::attention_tc_status(&t.status);
  if (!rc) rc = fovi::encode_rows(&tq, &t.q, a.q, a.q_sb, a.q_sl, a.q_sh, a.B, a.Lq, a.H, a.D, AT_M);
  if (!rc) rc = fovi::encode_rows(&tk, &t.k, a.k, a.k_sb, a.k_sl, a.k_sh, a.B, a.Lk, a.Hkv, a.D, KT);
  if (!rc) rc = fovi::encode_rows(&tv, &t.v, a.v, a.v_sb, a.v_sl, a.v_sh, a.B, a.Lk, a.Hkv, a.D, KT);
  if (rc) return rc;
  const int64_t blocks = (int64_t)((a.Lq + AT_M - 1) / AT_M) * a.H * a.B;
  if (blocks > INT_MAX) return FOVI_ERR_UNSUPPORTED;
  FOVI_CUDA(cudaFuncSetAttribute(attn_tc_forward_kernel<DC>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)F::SMEM));
  FOVI_CUDA(fovi::launch_pdl(attn_tc_forward_kernel<DC>, (int)blocks, AT_THREADS, F::SMEM, st, tq, tk, tv, t));
  return fovi::after_launch("attn_tc_forward_kernel");
}

}  // namespace

int fovi::encode_rows(CUtensorMap* m, TcView* view, const void* p, int64_t sb, int64_t sl, int64_t sh, int B, int L, int H, int D, int rows) {
  view->mul_h = H > 1 && sh > 0;
  view->mul_b = B > 1 && sb > 0;
  const uint64_t one = (uint64_t)(D + 7) / 8 * 16;        // the stride of an axis of extent 1 is never used
  const uint64_t dims[4] = {(uint64_t)D, (uint64_t)L, view->mul_h ? (uint64_t)H : 1, view->mul_b ? (uint64_t)B : 1};
  const uint64_t strides[3] = {L > 1 ? (uint64_t)sl * 2 : one, view->mul_h ? (uint64_t)sh * 2 : one, view->mul_b ? (uint64_t)sb * 2 : one};
  const uint32_t box[4] = {64, (uint32_t)rows, 1, 1};
  return fovi::encode_4d(m, p, dims, strides, box, true);
}

bool fovi::attention_tc_takes(const AttnArgs& a, int dtype, bool backward) {
  return dtype == FOVI_BF16 && a.D % 8 == 0 && a.D <= ATT_MAX_DIM && a.Lk > 0 && a.scale_log2 > 0.f && rows_ok(a.q, a.q_sb, a.q_sl, a.q_sh, a.B, a.Lq, a.H) &&
         rows_ok(a.k, a.k_sb, a.k_sl, a.k_sh, a.B, a.Lk, a.Hkv) && rows_ok(a.v, a.v_sb, a.v_sl, a.v_sh, a.B, a.Lk, a.Hkv) &&
         (backward ? rows_ok(a.dy, a.g_sb, a.g_sl, a.g_sh, a.B, a.Lq, a.H) && !((reinterpret_cast<uintptr_t>(a.o) | reinterpret_cast<uintptr_t>(a.dq) |
                                                                               reinterpret_cast<uintptr_t>(a.dk) | reinterpret_cast<uintptr_t>(a.dv)) & 15u)
                   : !(reinterpret_cast<uintptr_t>(a.out) & 15u));
}

int fovi::launch_attention_tc_forward(const AttnArgs& a, cudaStream_t st, bool selftest) {
  return a.D <= 64 ? forward<1>(a, st, selftest) : forward<2>(a, st, selftest);
}

int fovi::attention_tc_status(int** word) {
  FOVI_CUDA(cudaGetSymbolAddress(reinterpret_cast<void**>(word), g_status));
  return FOVI_OK;
}

int fovi::attention_tc_check(cudaStream_t st) {
  int site = 0;
  FOVI_CUDA(cudaMemcpyFromSymbolAsync(&site, g_status, sizeof(int), 0, cudaMemcpyDeviceToHost, st));
  FOVI_CUDA(cudaStreamSynchronize(st));
  if (!site) return FOVI_OK;
  const int zero = 0;
  FOVI_CUDA(cudaMemcpyToSymbolAsync(g_status, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, st));
  FOVI_CUDA(cudaStreamSynchronize(st));
  g_last_cuda_error = "attention: wait site " + std::to_string(site) + " gave up";
  return FOVI_ERR_DEVICE_TIMEOUT;
}
