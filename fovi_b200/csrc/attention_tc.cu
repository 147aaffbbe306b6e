// Cross attention on the tensor cores: bf16 q, k, v of up to 128 channels a head (a multiple of 8), 16-byte aligned rows.
//
// Forward.  One CTA per (128 queries, head, sample), three per SM (two above 64 channels); keys in tiles of 64.  Per tile
//   S = Q K^T     SS MMA, M = 128, N = 64, into tensor memory
//   P = 2^(scale log2(e) (S - m))     four warps, a thread per query: its row of S in registers, its running maximum and sum too; P goes to tensor memory as bf16
//   O += P V      TS MMA: P from tensor memory, the tile of V read MN-major, so nothing is transposed
// A fifth warp issues the tensor copies and both products.  S is given back as soon as its row is in registers, so the next tile's scores are computed while this one's exponentials
// are.  What bounds it are the exponentials (16 a clock and SM: 512 clocks a tile) and, as long as a warp's tile takes 1400 clocks in all (barriers, tensor memory and the
// maximum the rest), how many warps a scheduler has to choose from: three, with 128 registers each.  (A block's registers are given out evenly over the four schedulers: with two
// issuing warps, six in all, a third block would leave a thread 96.)  One exponential of eight is worked out on the multiply-add units (243 -> 230 us at 257 queries over 1028 keys,
// 256 x 6 heads; one of four: 233).  Measured: 256 queries over 4096 keys, 4 x 111 heads of 64 channels: 167 to 171 us, 700 TFLOP/s, 61 to 65 % of the exponential unit's rate; 4 x 74 heads of 128
// channels: 182 us, 874 TFLOP/s; one query over 2056 keys, 64 x 20 heads: 110 us, 6.1 TB/s.
// Few row tiles: their keys are cut into parts, one block each, joined by a second kernel (see splits_of).
// The reference value m of a row only moves when its maximum has risen
// by more than 8 (in base 2): P then stays below 2^8, bf16's relative rounding is the same at any size, and the pass over O that a move costs is rare.
// Masked keys: their scores are -inf by a select and their rows of V are set to zero in shared memory, so what they hold has no effect.  A warp whose
// 32 queries lie behind the last one skips the arithmetic.
#include <cuda_bf16.h>

#include "attention_tc.cuh"

using fovi::AttnArgs;
using fovi::AttnTcArgs;
using fovi::key_end;

namespace {

__device__ int g_status;           // wait site at which a kernel gave up, see fovi_attention_check: one word per device
constexpr int AT_THREADS = 160;
constexpr float AT_INF = __builtin_huge_valf();

// 2^x of two numbers x <= 8 on the multiply-add units: x = n + f with n whole and |f| <= 1/2 (Cody and Waite's reduction; n by adding 1.5 * 2^23), 2^f by a polynomial of degree 3 fitted
// with Remez' exchange (relative error 7.5e-5, a fiftieth of bf16's rounding), times 2^n.  Below -126 it stays 2^-126; not a number stays that.
__device__ __forceinline__ float2 ex2_fma(float2 x) {
  asm("max.NaN.f32 %0, %0, %2;\n max.NaN.f32 %1, %1, %2;" : "+f"(x.x), "+f"(x.y) : "f"(-126.f));
  const float2 t = add2(x, both(12582912.f)), f = fma2(add2(t, both(-12582912.f)), both(-1.f), x);
  float2 p = fma2(both(0.0551716685295105f), f, both(0.2426111251115799f));
  p = fma2(p, f, both(0.6932609677314758f));
  p = fma2(p, f, both(0.9999280571937561f));
  return mul2(p, make_float2(__int_as_float((__float_as_int(t.x) << 23) + 0x3f800000), __int_as_float((__float_as_int(t.y) << 23) + 0x3f800000)));
}

constexpr int KT = 64;             // keys of a tile

template <int DC> struct Fwd {                     // DC: 64-channel boxes of a row
  static constexpr int CTAS = DC == 1 ? 3 : 2;     // per SM
  static constexpr int NP = DC == 1 ? 1 : 2;       // places for P
  static constexpr int NK = DC == 1 ? 3 : 2, NV = NK;
  static constexpr uint32_t BOX = KT * 128u, TILE = DC * BOX, QBOX = AT_M * 128u, QTILE = DC * QBOX;
  static constexpr uint32_t SMEM = 1024 + 1024 + QTILE + (NK + NV) * TILE;
  // Tensor memory comes in powers of two.  One box: S and O in 128 columns and P in 32 of its own, so that three CTAs fit 512.
  static constexpr uint32_t COLS = DC == 1 ? 128 : 256, O_COL = DC == 1 ? 64 : 128, P_COLS = DC == 1 ? 32 : 0, P_COL = 64;
};

struct FwdHeader {
  uint64_t q_full, k_full[3], v_full[3], s_full, s_free, p_full[2], o_full, done, drain;
  uint32_t tmem_base, tmem_p;
  int abort_flag;
};

template <int DC>
__global__ void __launch_bounds__(AT_THREADS, Fwd<DC>::CTAS)
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
    for (int i = 0; i < 3; ++i) { mbar_init(smem_u32(&hdr->k_full[i]), 1); mbar_init(smem_u32(&hdr->v_full[i]), 1); }
    mbar_init(smem_u32(&hdr->s_full), 1); mbar_init(smem_u32(&hdr->s_free), 4);
    for (int i = 0; i < 2; ++i) mbar_init(smem_u32(&hdr->p_full[i]), 4);
    mbar_init(smem_u32(&hdr->o_full), 1); mbar_init(smem_u32(&hdr->done), 1); mbar_init(smem_u32(&hdr->drain), 1);
    hdr->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 4) {         // the small piece first: blocks that wait for the large one then hold next to nothing of what the others wait for
    if (F::P_COLS)
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&hdr->tmem_p)), "r"(32u) : "memory");
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&hdr->tmem_base)), "r"(F::COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int n_qt = (a.Lq + AT_M - 1) / AT_M, split = blockIdx.x % t.splits, block = blockIdx.x / t.splits;
  const int q0 = block % n_qt * AT_M, h = block / n_qt % a.H, b = block / n_qt / a.H, hk = h / a.group;
  const int end = key_end(a, b), share = ((end + KT - 1) / KT + t.splits - 1) / t.splits, first = split * share;       // tiles [first, first + tiles) of the keys
  const int tiles = min(max((end + KT - 1) / KT - first, 0), share);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = hdr->tmem_base, tmem_p = F::P_COLS ? hdr->tmem_p : tmem + F::P_COL;

  if (warp == 4) {
    // ------------------------------------------------------------ copies and MMAs (all lanes loop, one issues: see elect_one)
    const int dsteps = (a.D + 15) / 16;
    const uint32_t id_s = at_idesc(KT, false), id_o = at_idesc(dsteps * 16, true);
    const uint32_t u_sq = warp_uniform(sq), u_sk = warp_uniform(sk), u_sv = warp_uniform(sv), u_tmem = warp_uniform(tmem), u_p = warp_uniform(tmem_p);
    auto load_k = [&](int j) {
      const uint32_t bar = smem_u32(&hdr->k_full[j % F::NK]);
      mbar_expect_tx(bar, F::TILE);
      for (int c = 0; c < DC; ++c) tma_load_4d(u_sk + j % F::NK * F::TILE + c * F::BOX, &tm_k, bar, 64 * c, (first + j) * KT, hk * t.k.mul_h, b * t.k.mul_b);
    };
    auto load_v = [&](int j) {
      const uint32_t bar = smem_u32(&hdr->v_full[j % F::NV]);
      mbar_expect_tx(bar, F::TILE);
      for (int c = 0; c < DC; ++c) tma_load_4d(u_sv + j % F::NV * F::TILE + c * F::BOX, &tm_v, bar, 64 * c, (first + j) * KT, hk * t.v.mul_h, b * t.v.mul_b);
    };
    auto scores = [&](int j) {
      if (!at_wait(smem_u32(&hdr->k_full[j % F::NK]), j / F::NK & 1, abort_flag, t.status, 4, t.wait_limit)) return false;
      if (j > 0 && !at_wait(smem_u32(&hdr->s_free), (j - 1) & 1, abort_flag, t.status, 5, t.wait_limit)) return false;
      tc_fence_after();
      mma_rows<DC>(u_tmem, u_sq, F::QBOX, u_sk + warp_uniform(j % F::NK) * F::TILE, F::BOX, id_s);
      if (elect_one()) {
        tc_commit(smem_u32(&hdr->s_full));      // and with it the product of tile j - 2, which this thread issued before
        if (j > 0 && j - 1 + F::NK < tiles) load_k(j - 1 + F::NK);      // the scores of tile j - 1 were read: its K is done with
      }
      __syncwarp();
      return true;
    };
    bool ok = true;
    if (tiles > 0) {
      if (!t.skip_loads && elect_one()) {
        const uint32_t qf = smem_u32(&hdr->q_full);
        mbar_expect_tx(qf, F::QTILE);
        for (int c = 0; c < DC; ++c) tma_load_4d(u_sq + c * F::QBOX, &tm_q, qf, 64 * c, q0, h * t.q.mul_h, b * t.q.mul_b);
        for (int j = 0; j < F::NK && j < tiles; ++j) { load_k(j); load_v(j); }
      }
      __syncwarp();
      ok = at_wait(smem_u32(&hdr->q_full), 0, abort_flag, t.status, 3, t.wait_limit) && scores(0);
    }
    for (int j = 0; j < tiles && ok; ++j) {
      if (j + 1 < tiles) ok = scores(j + 1);
      ok = ok && at_wait(smem_u32(&hdr->v_full[j % F::NV]), j / F::NV & 1, abort_flag, t.status, 6, t.wait_limit);
      ok = ok && at_wait(smem_u32(&hdr->p_full[j & 1]), j >> 1 & 1, abort_flag, t.status, 7, t.wait_limit);
      // (waited for in front of the next product: behind it this phase of the barrier could not be told from the one after the next)
      const bool more_v = j > 0 && j - 1 + F::NV < tiles;
      if (more_v) ok = ok && at_wait(smem_u32(&hdr->o_full), (j - 1) & 1, abort_flag, t.status, 2, t.wait_limit);
      if (!ok) break;
      tc_fence_after();
      mma_mix(u_tmem + F::O_COL, u_p + (F::NP == 2 ? (j & 1) * (KT / 2) : 0), u_sv + warp_uniform(j % F::NV) * F::TILE, F::BOX, KT / 16, id_o, j > 0);
      if (elect_one()) {
        tc_commit(smem_u32(&hdr->o_full));
        if (j + 1 == tiles) tc_commit(smem_u32(&hdr->done));
        if (more_v) load_v(j - 1 + F::NV);                 // the product before this one is done, and its V with it
      }
      __syncwarp();
    }
    if (*abort_flag) {
      if (elect_one()) {                   // no MMA may still be reading shared memory or writing tensor memory
        tc_commit(smem_u32(&hdr->drain));
        for (uint32_t it = 0; it < (1u << 20); ++it)
          if (mbar_try_wait(smem_u32(&hdr->drain), 0)) break;
      }
      for (int i = 0; i < 64; ++i) __nanosleep(1000);      // copies in flight get time to land before the block leaves its shared memory
    }
  } else {
    // ------------------------------------------------------------ softmax: thread = query
    const int row = q0 + threadIdx.x;
    const bool idle = q0 + warp * 32 >= a.Lq;          // no query in this warp
    const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16), lanes_p = tmem_p + ((uint32_t)(warp * 32) << 16);
    const uint8_t* mask = a.mask ? a.mask + (int64_t)b * a.Lk : nullptr;
    const float c = a.scale_log2;
    float m = -AT_INF;                 // the row's reference value, in units of S
    float2 l[4] = {};                  // its sum, in eight parts: additions that do not wait for one another
    bool ok = true;
    for (int j = 0; j < tiles; ++j) {
      uint32_t bits[KT / 32];
      const int key0 = (first + j) * KT;
      bool whole = !mask && key0 + KT <= end;
      if (!whole) {
        whole = true;
#pragma unroll
        for (int i = 0; i < KT / 32; ++i) { bits[i] = key_bits(a, mask, key0 + 32 * i, end, lane); whole = whole && bits[i] == 0xffffffffu; }
      }
      ok = at_wait(smem_u32(&hdr->s_full), j & 1, abort_flag, t.status, 8, t.wait_limit);
      if (!ok) break;
      tc_fence_after();
      float x[KT];
      if (!idle) {
#pragma unroll
        for (int i = 0; i < KT; i += 32) tc_ld32(lanes + i, reinterpret_cast<uint32_t*>(x) + i);
        tc_ld_wait();
        tc_loaded<KT>(reinterpret_cast<uint32_t*>(x));
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&hdr->s_free));
      bool move = false;
      float m_new = m;
      if (!idle) {
        if (!whole) {
#pragma unroll
          for (int i = 0; i < KT; ++i) x[i] = bits[i >> 5] >> (i & 31) & 1u ? x[i] : -AT_INF;
        }
        float top[4] = {m, m, m, m};
#pragma unroll
        for (int i = 0; i < KT; i += 8) {
#pragma unroll
          for (int e = 0; e < 4; ++e) top[e] = max3(top[e], x[i + 2 * e], x[i + 2 * e + 1]);
        }
        m_new = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        move = (m_new - m) * c > 8.f;
      }
      // The place for P.  One: the product before this one has to be done, and every warp waits for it in every tile.  Two: this tile's scores say that the product before the last is
      // done and that every warp has arrived for it; a warp can be ahead of another by a tile, never by the two that would let it arrive twice at the barriers, which come in pairs.
      if (F::NP == 1 && j > 0 && !at_wait(smem_u32(&hdr->o_full), (j - 1) & 1, abort_flag, t.status, 9, t.wait_limit)) { ok = false; break; }
      if (__any_sync(0xffffffffu, move)) {
        const float f = move ? ex2((m - m_new) * c) : 1.f;
        if (move) m = m_new;
#pragma unroll
        for (int e = 0; e < 4; ++e) l[e] = mul2(l[e], make_float2(f, f));
        if (F::NP == 2 && j > 0 && !at_wait(smem_u32(&hdr->o_full), (j - 1) & 1, abort_flag, t.status, 9, t.wait_limit)) { ok = false; break; }
        if (j > 0) {                    // the product with the previous P is done: O is this thread's
          tc_fence_after();
#pragma unroll 1
          for (int o = 0; o < DC * 64; o += 16) {
            uint32_t r[16];
            tc_ld16(lanes + F::O_COL + o, r);
            tc_ld_wait();
            tc_loaded<16>(r);
#pragma unroll
            for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * f);
            tc_st16(lanes + F::O_COL + o, r);
          }
        }
      }
      if (!idle) {
        const float mc = m == -AT_INF ? 0.f : m * c;      // no key yet: every exponent is -inf
#pragma unroll
        for (int p = 0; p < KT; p += 32) {
          uint32_t w[16];
#pragma unroll
          for (int i = p; i < p + 32; i += 2) {
            const float2 e = fma2(make_float2(x[i], x[i + 1]), make_float2(c, c), make_float2(-mc, -mc));
            const float2 y = i / 2 % 8 == 3 ? ex2_fma(e) : make_float2(ex2(e.x), ex2(e.y));      // one pair of eight beside the exponential unit
            l[i / 2 % 4] = add2(l[i / 2 % 4], y);
            w[(i - p) >> 1] = pack_bf16(y.x, y.y);
          }
          tc_st16(lanes_p + (F::NP == 2 ? (j & 1) * (KT / 2) : 0) + p / 2, w);
        }
      }
      if (!whole) {                     // rows of V that must not be read: a zero weight times what they hold need not be zero
        ok = at_wait(smem_u32(&hdr->v_full[j % F::NV]), (j / F::NV) & 1, abort_flag, t.status, 10, t.wait_limit);
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
      if (lane == 0) mbar_arrive(smem_u32(&hdr->p_full[j & 1]));
    }
    if (ok && tiles > 0) ok = at_wait(smem_u32(&hdr->done), 0, abort_flag, t.status, 11, t.wait_limit);
    if (ok && !idle) {
      tc_fence_after();
      const bool none = m == -AT_INF;
      const float2 l2 = add2(add2(l[0], l[1]), add2(l[2], l[3]));
      const float sum = l2.x + l2.y, inv = none ? 0.f : 1.f / sum;
      // `none` also holds for a row of scores that are all not a number; its sum is not a number then, and so is its result
      const bool zero = none && !(sum != sum);
      const int64_t at = ((int64_t)b * a.Lq + row) * a.H + h, rows = (int64_t)a.B * a.Lq * a.H;
      __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + at * a.D;
      float* part = t.part_o + (split * rows + at) * a.D;
#pragma unroll
      for (int o = 0; o < DC * 64; o += 32) {
        uint32_t r[32];
        if (tiles > 0) { tc_ld32(lanes + F::O_COL + o, r); tc_ld_wait(); tc_loaded<32>(r); }
        if (row < a.Lq) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            if (o + 8 * g < a.D) {
              if (t.splits > 1) {            // a part of the keys: float32, for the join
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                  float u[4];
#pragma unroll
                  for (int e = 0; e < 4; ++e) u[e] = zero ? 0.f : none ? sum : __uint_as_float(r[8 * g + 4 * i + e]) * inv;
                  *reinterpret_cast<float4*>(part + o + 8 * g + 4 * i) = make_float4(u[0], u[1], u[2], u[3]);
                }
                continue;
              }
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
      const float lse = zero ? AT_INF : m * c + log2f(sum);
      if (row < a.Lq) {
        if (t.splits > 1) t.part_lse[split * rows + at] = lse;
        else if (a.lse) a.lse[((int64_t)b * a.H + h) * a.Lq + row] = lse;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 4) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(F::COLS) : "memory");
  if (warp == 4 && F::P_COLS) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_p), "r"(32u) : "memory");
}

// The parts of a row over the splits of its keys, weighted with the parts' sums, added in their order.  A thread for four channels.
__global__ void __launch_bounds__(256) attn_join_kernel(const AttnTcArgs t) {
  const AttnArgs& a = t.a;
  const int per = a.D / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, rows = (int64_t)a.B * a.Lq * a.H, row = i / per;
  if (row >= rows) return;
  const int d = (int)(i - row * per) * 4;
  float top = -AT_INF;                    // a part without a key has +inf in place of its logarithm
  for (int s = 0; s < t.splits; ++s) {
    const float v = __ldg(t.part_lse + s * rows + row);
    top = v == AT_INF ? top : v != v ? v : fmaxf(top, v);
  }
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
  for (int s = 0; s < t.splits; ++s) {
    const float v = __ldg(t.part_lse + s * rows + row);
    if (v == AT_INF) continue;
    const float w = exp2f(v - top);
    const float4 p = __ldg(reinterpret_cast<const float4*>(t.part_o + (s * rows + row) * a.D + d));
    o.x = fmaf(w, p.x, o.x); o.y = fmaf(w, p.y, o.y); o.z = fmaf(w, p.z, o.z); o.w = fmaf(w, p.w, o.w);
    sum += w;
  }
  const bool none = top == -AT_INF;
  const float inv = none ? 0.f : 1.f / sum;
  uint2 w;
  w.x = pack_bf16(o.x * inv, o.y * inv); w.y = pack_bf16(o.z * inv, o.w * inv);
  *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + row * a.D + d) = w;
  if (a.lse && d == 0) {
    const int h = (int)(row % a.H);
    const int64_t bl = row / a.H, b = bl / a.Lq;
    a.lse[(b * a.H + h) * a.Lq + (bl - b * a.Lq)] = none ? AT_INF : top + log2f(sum);
  }
}

// ------------------------------------------------------------------------------------------------------------ host
bool rows_ok(const void* p, int64_t sb, int64_t sl, int64_t sh, int B, int L, int H) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (L == 1 || (sl > 0 && sl % 8 == 0)) && (H == 1 || sh % 8 == 0) && (B == 1 || sb % 8 == 0) &&
         sl < (int64_t)1 << 38 && sh < (int64_t)1 << 38 && sb < (int64_t)1 << 38;
}

// Into how many parts the keys of a row tile are cut, so that the blocks fill the SMs: the number for which the rounds of blocks, each as long as its tiles and about six more for a block's
// beginning and end, are shortest.  More than one part also costs the join, a launch and a pass over the parts: about eight tiles.
int splits_of(int B, int Lq, int Lk, int H, int D) {
  const int64_t blocks = (int64_t)((Lq + AT_M - 1) / AT_M) * H * B, slots = (int64_t)fovi::sm_count() * (D <= 64 ? Fwd<1>::CTAS : Fwd<2>::CTAS);
  const int tiles = (Lk + KT - 1) / KT;
  int best = 1;
  int64_t least = INT64_MAX;
  for (int s = 1; s <= 32 && s <= tiles; ++s) {
    const int64_t time = (blocks * s + slots - 1) / slots * ((tiles + s - 1) / s + 6) + (s > 1 ? 8 : 0);
    if (time < least) { least = time; best = s; }
  }
  return best;
}

template <int DC>
int forward(const AttnArgs& a, void* work, cudaStream_t st, bool selftest) {
  using F = Fwd<DC>;
  CUtensorMap tq, tk, tv;
  AttnTcArgs t = {};
  t.splits = work ? splits_of(a.B, a.Lq, a.Lk, a.H, a.D) : 1;
  t.part_o = static_cast<float*>(work);
  t.part_lse = t.part_o + (int64_t)t.splits * a.B * a.Lq * a.H * a.D;
  t.a = a;
  t.wait_limit = selftest ? 4096u : WAIT_LIMIT;
  t.skip_loads = selftest;
  int rc = fovi::attention_tc_status(&t.status);
  if (!rc) rc = fovi::encode_rows(&tq, &t.q, a.q, a.q_sb, a.q_sl, a.q_sh, a.B, a.Lq, a.H, a.D, AT_M);
  if (!rc) rc = fovi::encode_rows(&tk, &t.k, a.k, a.k_sb, a.k_sl, a.k_sh, a.B, a.Lk, a.Hkv, a.D, KT);
  if (!rc) rc = fovi::encode_rows(&tv, &t.v, a.v, a.v_sb, a.v_sl, a.v_sh, a.B, a.Lk, a.Hkv, a.D, KT);
  if (rc) return rc;
  const int64_t blocks = (int64_t)((a.Lq + AT_M - 1) / AT_M) * a.H * a.B * t.splits, join = ((int64_t)a.B * a.Lq * a.H * (a.D / 4) + 255) / 256;
  if (blocks > INT_MAX || join > INT_MAX) return FOVI_ERR_UNSUPPORTED;
  FOVI_CUDA(cudaFuncSetAttribute(attn_tc_forward_kernel<DC>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)F::SMEM));
  FOVI_CUDA(fovi::launch_pdl(attn_tc_forward_kernel<DC>, (int)blocks, AT_THREADS, F::SMEM, st, tq, tk, tv, t));
  rc = fovi::after_launch("attn_tc_forward_kernel");
  if (rc || t.splits == 1) return rc;
  attn_join_kernel<<<(int)join, 256, 0, st>>>(t);
  return fovi::after_launch("attn_join_kernel");
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

int64_t fovi::attention_tc_forward_bytes(int B, int Lq, int Lk, int H, int D) {
  const int s = splits_of(B, Lq, Lk, H, D);
  return s == 1 ? 0 : (int64_t)s * B * Lq * H * (D + 1) * 4;
}

int fovi::launch_attention_tc_forward(const AttnArgs& a, void* work, cudaStream_t st, bool selftest) {
  return a.D <= 64 ? forward<1>(a, work, st, selftest) : forward<2>(a, work, st, selftest);
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
