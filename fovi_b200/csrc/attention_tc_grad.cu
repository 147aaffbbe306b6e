// Gradients of cross attention on the tensor cores (bf16, see attention_tc.cu for the shapes).
//   p = 2^(scale log2(e) s - lse),  ds = p * (dp - delta),  s = q k^T, dp = dy v^T
//   dq = scale * sum over keys of ds k          dv = sum over queries of p dy,   dk = scale * sum over queries of ds q
// Two kernels of one form: a CTA owns 128 rows (queries for dq; keys for dk and dv), whose two operand tiles stay in shared memory, and goes over tiles of CT columns
// (the keys; the queries of all heads that read the state head).  Per tile
//   S = R1 C1^T, dP = R2 C2^T          SS MMAs, M = 128, N = CT, into tensor memory; for dk and dv these are the transposed scores, rows = keys
//   P, dS                              eight warps, a thread per row and half the columns: registers, then back to tensor memory as bf16
//   acc1 += dS C1 (dq, dk),  acc2 += P C2 (dv; P C1 for dq)          TS MMAs, the column tiles read MN-major: nothing is transposed, nothing goes through shared memory
// Each gradient is summed by one CTA in a fixed order: no atomics, the same bits every time, no float32 buffer of dq, for 8 products instead of 5.
// The eighth, sum p k, is for delta: taken from the rounded result it is off by some 0.2 % of a dp's size, the same for all of a row's keys, which where a row's weight lies on few keys
// was a tenth to a fifth of dq's and dk's whole error.  The row's sum of ds says how far it is off.
// One CTA per SM with all 512 columns of tensor memory, over many row tiles (persistent).  Beside the eight warps one issues the scores, one the products, one the copies in and one the
// copies out: a single MMA warp spent 2000 clocks a tile on its barriers and on issuing, one after the other, where the tensor cores have 800 to 1100 of work.
// The next tile's scores are computed while this one's elements are worked on, and the next row tile's operands arrive meanwhile.  Results go through the row tile's own operand buffers, which the scores are done
// with, and out as tensor copies: stored from registers, 16 bytes of a row per thread, they took half the time of dk and dv (716 us with, 400 without them, 4 x 111 heads, 256 over 4096).
// A last tile of fewer columns costs only its own (N and the steps over its columns follow).
// Rows of K whose key is masked are set to zero in shared memory in front of dS K; for dk and dv a masked key is a row, whose results are zeros by a select.
// Measured with the rows' statistics (us; 257 queries over 1028 keys, 256 x 6 heads of 64 channels; 256 over 4096, 4 x 111 heads): dq 391 and 236, dk and dv 444 and 363.  Time stamps
// of one warp of dq at a tile of 128 x 128 (period 2000 clocks; taken before masks became a step of their own): elements 1360, waits for the scores 180 and for the last products 200,
// stores 140; the exponential unit needs 1024 for the two warps of a scheduler.
// A mask is applied to a whole chunk of scores in front of the arithmetic, and only where one is: selects at each p and ds cost every tile (ALU pipe 50 %, now 20; dq 405 and 243 us).
// 16 columns at a time, the next on their way, was slower (dq 211 -> 236 us, 4 x 111 heads, an earlier form).
#include <cuda_bf16.h>

#include "attention_tc.cuh"
#include "row_turns.cuh"

using fovi::AttnArgs;
using fovi::AttnTcArgs;
using fovi::key_end;
using fovi::RowTurn;

namespace {

constexpr int EW_WARPS = 8, GR_THREADS = (EW_WARPS + 4) * 32;        // then the warps of the scores, the products, the copies in, the copies out
constexpr int SCORES = EW_WARPS, PRODUCTS = EW_WARPS + 1, LOADS = EW_WARPS + 2, STORES = EW_WARPS + 3;
constexpr float AT_INF = __builtin_huge_valf();

template <int DC> struct Grad {
  static constexpr int CT = DC == 1 ? 128 : 64, HALF = CT / 2;       // columns of a tile, of a thread
  static constexpr int NS = DC == 1 ? 4 : 3;                         // column tiles in flight
  static constexpr uint32_t RBOX = AT_M * 128u, RTILE = DC * RBOX, CBOX = CT * 128u, CTILE = DC * CBOX;
  static constexpr uint32_t ROWS = 4 * RTILE;                        // two row tiles of two operands
  static constexpr uint32_t SMEM = 1024 + ROWS + NS * 2 * CTILE + NS * 2 * CT * 4 + 256;         // slack for the alignment, tiles, row statistics, barriers
  static constexpr uint32_t DP = CT, P = 2 * CT, DS = 2 * CT + CT / 2, ACC1 = DC == 1 ? 384 : 256, ACC2 = ACC1 + 64 * DC;
};

struct GradHeader {
  uint64_t row_full[2], row_empty[2], full[4], empty[4], s_full, s_free, p_full, mixed, acc_full, acc_free, summed, staged[2], drain[2];
  uint32_t tmem_base;
  int abort_flag;
};

struct GradArgs {
  AttnTcArgs t;
  const float *nl, *nd;        // [B, H, pitch]: -lse and -delta, -inf and 0 behind the last query
  float* nd_out;               // dq: -delta without its error
  int pitch, items, tiles;     // tiles: row tiles of a head
};

struct Item { int row0, h, b, end, n; };     // h: query head (dq) or state head (dk, dv); n: column tiles

template <int DC, bool KEYS>
__device__ __forceinline__ Item item_at(const GradArgs& g, int i) {
  const AttnArgs& a = g.t.a;
  const int heads = KEYS ? a.Hkv : a.H;
  Item it;
  it.row0 = i % g.tiles * AT_M; it.h = i / g.tiles % heads; it.b = i / g.tiles / heads;
  it.end = key_end(a, it.b);
  it.n = KEYS ? (it.row0 < it.end ? a.group * ((a.Lq + Grad<DC>::CT - 1) / Grad<DC>::CT) : 0) : (it.end + Grad<DC>::CT - 1) / Grad<DC>::CT;
  return it;
}

// (row tile, column tile) pairs in the order in which every role meets them; row tiles without columns are passed over.
template <int DC, bool KEYS>
struct Walk {
  int i, j;
  RowTurn row;                 // counts the row tiles with columns
  Item it;
  __device__ __forceinline__ explicit Walk(const GradArgs& g) : i(blockIdx.x), j(0) { settle(g); }
  __device__ __forceinline__ void settle(const GradArgs& g) {
    for (; i < g.items; i += gridDim.x) {
      it = item_at<DC, KEYS>(g, i);
      if (it.n > 0) return;
    }
  }
  __device__ __forceinline__ bool more(const GradArgs& g) const { return i < g.items; }
  __device__ __forceinline__ void next(const GradArgs& g) {
    if (++j < it.n) return;
    next_row(g);
  }
  __device__ __forceinline__ void next_row(const GradArgs& g) {
    j = 0; row.next(); i += gridDim.x;
    settle(g);
  }
};

// Columns of tile j: first one, and how many there are.
template <int DC, bool KEYS>
__device__ __forceinline__ int columns(const AttnArgs& a, const Item& it, int j, int& c0, int& h) {
  constexpr int CT = Grad<DC>::CT;
  const int per = KEYS ? (a.Lq + CT - 1) / CT : it.n;
  const int q = KEYS ? j / per : 0;
  c0 = (j - q * per) * CT;
  h = KEYS ? it.h * a.group + q : it.h;
  return min(CT, (KEYS ? a.Lq : it.end) - c0);
}

template <int DC, bool KEYS>
__global__ void __launch_bounds__(GR_THREADS, 1)
attn_tc_grad_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                    const __grid_constant__ CUtensorMap tm_g, const __grid_constant__ CUtensorMap tm_1, const __grid_constant__ CUtensorMap tm_2, const GradArgs g) {
  using G = Grad<DC>;
  constexpr int CT = G::CT, HALF = G::HALF;
  const AttnTcArgs& t = g.t;
  const AttnArgs& a = t.a;
  extern __shared__ unsigned char smem_raw[];
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  const uint32_t srow = base, scol = srow + G::ROWS, sstat = scol + G::NS * 2 * G::CTILE;
  static_assert(sizeof(GradHeader) <= 256 && G::SMEM <= 232448, "shared memory of a block");
  GradHeader* hdr = reinterpret_cast<GradHeader*>(smem_raw + (sstat - raw) + G::NS * 2 * CT * 4);
  volatile int* abort_flag = &hdr->abort_flag;
  int* status = t.status;
  const int warp = warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) { mbar_init(smem_u32(&hdr->row_full[i]), 1); mbar_init(smem_u32(&hdr->row_empty[i]), 1); mbar_init(smem_u32(&hdr->staged[i]), EW_WARPS); mbar_init(smem_u32(&hdr->drain[i]), 1); }
    for (int i = 0; i < 4; ++i) { mbar_init(smem_u32(&hdr->full[i]), 1); mbar_init(smem_u32(&hdr->empty[i]), 1); }
    mbar_init(smem_u32(&hdr->s_full), 1); mbar_init(smem_u32(&hdr->s_free), EW_WARPS); mbar_init(smem_u32(&hdr->p_full), EW_WARPS);
    mbar_init(smem_u32(&hdr->mixed), 1); mbar_init(smem_u32(&hdr->acc_full), 1); mbar_init(smem_u32(&hdr->acc_free), EW_WARPS);
    mbar_init(smem_u32(&hdr->summed), EW_WARPS);
    hdr->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == SCORES) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&hdr->tmem_base)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = hdr->tmem_base;

  if (warp == LOADS) {
    // ------------------------------------------------------------ copies in
    if (lane == 0 && !t.skip_loads) {
      uint32_t s = 0, sp = 0;
      for (Walk<DC, KEYS> w(g); w.more(g); w.next(g)) {
        if (w.j == 0) {
          const uint32_t f = w.row.buffer(), fp = w.row.parity(), bar = smem_u32(&hdr->row_full[f]), dst = srow + f * 2 * G::RTILE;
          if (!mbar_wait(smem_u32(&hdr->row_empty[f]), fp ^ 1u, abort_flag, status, 21, t.wait_limit)) break;
          mbar_expect_tx(bar, 2 * G::RTILE);
          for (int c = 0; c < DC; ++c) {
            if (KEYS) {
              tma_load_4d(dst + c * G::RBOX, &tm_k, bar, 64 * c, w.it.row0, w.it.h * t.k.mul_h, w.it.b * t.k.mul_b);
              tma_load_4d(dst + G::RTILE + c * G::RBOX, &tm_v, bar, 64 * c, w.it.row0, w.it.h * t.v.mul_h, w.it.b * t.v.mul_b);
            } else {
              tma_load_4d(dst + c * G::RBOX, &tm_q, bar, 64 * c, w.it.row0, w.it.h * t.q.mul_h, w.it.b * t.q.mul_b);
              tma_load_4d(dst + G::RTILE + c * G::RBOX, &tm_g, bar, 64 * c, w.it.row0, w.it.h * t.g.mul_h, w.it.b * t.g.mul_b);
            }
          }
        }
        int c0, h;
        columns<DC, KEYS>(a, w.it, w.j, c0, h);
        if (!mbar_wait(smem_u32(&hdr->empty[s]), sp ^ 1u, abort_flag, status, 22, t.wait_limit)) break;
        const uint32_t bar = smem_u32(&hdr->full[s]), dst = scol + s * 2 * G::CTILE;
        mbar_expect_tx(bar, 2 * G::CTILE + (KEYS ? 2 * CT * 4 : 0));
        for (int c = 0; c < DC; ++c) {
          if (KEYS) {
            tma_load_4d(dst + c * G::CBOX, &tm_q, bar, 64 * c, c0, h * t.q.mul_h, w.it.b * t.q.mul_b);
            tma_load_4d(dst + G::CTILE + c * G::CBOX, &tm_g, bar, 64 * c, c0, h * t.g.mul_h, w.it.b * t.g.mul_b);
          } else {
            tma_load_4d(dst + c * G::CBOX, &tm_k, bar, 64 * c, c0, h / a.group * t.k.mul_h, w.it.b * t.k.mul_b);
            tma_load_4d(dst + G::CTILE + c * G::CBOX, &tm_v, bar, 64 * c, c0, h / a.group * t.v.mul_h, w.it.b * t.v.mul_b);
          }
        }
        if (KEYS) {
          const int64_t at = ((int64_t)w.it.b * a.H + h) * g.pitch + c0;
          bulk_load(sstat + s * 2 * CT * 4, g.nl + at, CT * 4, bar);
          bulk_load(sstat + s * 2 * CT * 4 + CT * 4, g.nd + at, CT * 4, bar);
        }
        if (++s == G::NS) { s = 0; sp ^= 1u; }
      }
      if (*abort_flag)      // copies in flight get time to land before the block leaves its shared memory
        for (int i = 0; i < 64; ++i) __nanosleep(1000);
    }
  } else if (warp == SCORES) {
    // ------------------------------------------------------------ S and dP (the MMA warps loop with all lanes, one issues: see elect_one)
    const uint32_t u_srow = warp_uniform(srow), u_scol = warp_uniform(scol), u_tmem = warp_uniform(tmem);
    uint32_t s = 0, sp = 0, n = 0;
    for (Walk<DC, KEYS> w(g); w.more(g); w.next(g), ++n) {
      const uint32_t f = w.row.buffer();
      if (w.j == 0 && !at_wait(smem_u32(&hdr->row_full[f]), w.row.parity(), abort_flag, status, 23, t.wait_limit)) break;
      if (!at_wait(smem_u32(&hdr->full[s]), sp, abort_flag, status, 24, t.wait_limit)) break;
      if (n > 0 && !at_wait(smem_u32(&hdr->s_free), (n - 1) & 1, abort_flag, status, 25, t.wait_limit)) break;
      tc_fence_after();
      int c0, h;
      const int cols = warp_uniform((columns<DC, KEYS>(a, w.it, w.j, c0, h) + 15) / 16 * 16);
      const uint32_t rows = warp_uniform(u_srow + f * 2 * G::RTILE), tile = warp_uniform(u_scol + s * 2 * G::CTILE), id = at_idesc(0, false) | ((uint32_t)(cols >> 3) << 17);
      mma_rows<DC>(u_tmem, rows, G::RBOX, tile, G::CBOX, id);
      mma_rows<DC>(u_tmem + G::DP, rows + G::RTILE, G::RBOX, tile + G::CTILE, G::CBOX, id);
      if (elect_one()) tc_commit(smem_u32(&hdr->s_full));
      __syncwarp();
      if (++s == G::NS) { s = 0; sp ^= 1u; }
    }
    // No MMA may still be reading shared memory or writing tensor memory when the block leaves.  A commit covers its own warp's MMAs only, so each of the two warps has a barrier for this:
    // on one for both, the first to arrive would let the other go with MMAs in flight, and two arrivals before a look would look like none.
    if (*abort_flag && elect_one()) {
      tc_commit(smem_u32(&hdr->drain[0]));
      for (uint32_t it = 0; it < (1u << 20); ++it)
        if (mbar_try_wait(smem_u32(&hdr->drain[0]), 0)) break;
    }
  } else if (warp == PRODUCTS) {
    // ------------------------------------------------------------ the accumulators
    const uint32_t id_acc = at_idesc((a.D + 15) / 16 * 16, true);
    const uint32_t u_scol = warp_uniform(scol), u_tmem = warp_uniform(tmem);
    uint32_t s = 0, sp = 0, n = 0;
    for (Walk<DC, KEYS> w(g); w.more(g); w.next(g), ++n) {
      if (!at_wait(smem_u32(&hdr->full[s]), sp, abort_flag, status, 26, t.wait_limit)) break;
      if (w.j == 0 && w.row.seq > 0 && !at_wait(smem_u32(&hdr->acc_free), (w.row.seq - 1) & 1, abort_flag, status, 27, t.wait_limit)) break;
      if (!at_wait(smem_u32(&hdr->p_full), n & 1, abort_flag, status, 32, t.wait_limit)) break;
      tc_fence_after();
      int c0, h;
      const int steps = warp_uniform((columns<DC, KEYS>(a, w.it, w.j, c0, h) + 15) / 16);
      const uint32_t tile = warp_uniform(u_scol + s * 2 * G::CTILE);
      const bool more = warp_uniform(w.j) > 0;
#pragma unroll
      for (int q = 0; q < CT / 64; ++q) {         // 64 columns at a time
        if (!KEYS && !a.dq) break;                // for delta alone
        mma_mix(u_tmem + G::ACC2, u_tmem + G::P + q * 32, tile + (KEYS ? G::CTILE : 0u) + q * 8192, G::CBOX, steps - 4 * q, id_acc, more || q);
        mma_mix(u_tmem + G::ACC1, u_tmem + G::DS + q * 32, tile + q * 8192, G::CBOX, steps - 4 * q, id_acc, more || q);
      }
      if (elect_one()) {
        tc_commit(smem_u32(&hdr->empty[s]));
        tc_commit(smem_u32(&hdr->mixed));
        if (w.j + 1 == w.it.n) tc_commit(smem_u32(&hdr->acc_full));
      }
      __syncwarp();
      if (++s == G::NS) { s = 0; sp ^= 1u; }
    }
    if (*abort_flag && elect_one()) {
      tc_commit(smem_u32(&hdr->drain[1]));
      for (uint32_t it = 0; it < (1u << 20); ++it)
        if (mbar_try_wait(smem_u32(&hdr->drain[1]), 0)) break;
    }
  } else if (warp == STORES) {
    // ------------------------------------------------------------ copies out
    for (Walk<DC, KEYS> w(g); w.more(g); w.next_row(g)) {
      const uint32_t f = w.row.buffer(), from = srow + f * 2 * G::RTILE;
      if (!at_wait(smem_u32(&hdr->staged[f]), w.row.parity(), abort_flag, status, 33, t.wait_limit)) break;
      if (elect_one()) {
        for (int c = 0; c < DC; ++c) {
          if (KEYS ? a.dk : a.dq) tma_store_4d(&tm_1, from + c * G::RBOX, 64 * c, w.it.row0, w.it.h, w.it.b);
          if (KEYS) tma_store_4d(&tm_2, from + G::RTILE + c * G::RBOX, 64 * c, w.it.row0, w.it.h, w.it.b);
        }
        bulk_commit_and_read();                // the buffers may be filled again
        mbar_arrive(smem_u32(&hdr->row_empty[f]));
      }
      __syncwarp();
    }
  } else {
    // ------------------------------------------------------------ elements: thread = row, half the columns
    const int r = (warp & 3) * 32 + lane, half = warp >> 2;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const float c = a.scale_log2;
    uint32_t n = 0, slot = 0, sphase = 0;
    RowTurn turn;
    bool ok = true;
    for (int i = blockIdx.x; ok && i < g.items; i += gridDim.x) {
      const Item it = item_at<DC, KEYS>(g, i);
      const int row = it.row0 + r;
      const bool idle = it.row0 + (warp & 3) * 32 >= (KEYS ? it.end : a.Lq);
      const uint8_t* mask = a.mask ? a.mask + (int64_t)it.b * a.Lk : nullptr;
      float nl = 0.f, nd = 0.f;
      bool row_ok = true;
      if (KEYS) {
        row_ok = row < it.end && (!mask || __ldg(mask + row));
      } else if (row < g.pitch) {
        const int64_t at = ((int64_t)it.b * a.H + it.h) * g.pitch + row;
        nl = __ldg(g.nl + at); nd = __ldg(g.nd + at);
      }
      float2 rest[2] = {};                   // dq: the sum of the row's ds, of this thread's columns
      for (int j = 0; j < it.n; ++j, ++n) {
        int c0, h;
        const int cols = columns<DC, KEYS>(a, it, j, c0, h);
        const int first = half * HALF;
        uint32_t bits[HALF / 32];
        bool whole = KEYS || (!mask && cols == CT);
        if (!whole) {
          whole = true;
#pragma unroll
          for (int e = 0; e < HALF / 32; ++e) { bits[e] = key_bits(a, mask, c0 + first + 32 * e, it.end, lane); whole = whole && bits[e] == 0xffffffffu; }
        }
        ok = at_wait(smem_u32(&hdr->s_full), n & 1, abort_flag, status, 28, t.wait_limit);
        if (ok && KEYS) ok = at_wait(smem_u32(&hdr->full[slot]), sphase, abort_flag, status, 29, t.wait_limit);     // (done: the scores needed it too)
        if (!ok) break;
        tc_fence_after();
        const float* st = reinterpret_cast<const float*>(smem_raw + (sstat - raw) + slot * 2 * CT * 4) + first;
#pragma unroll
        for (int e = 0; e < HALF; e += 32) {          // 32 columns at a time: all of them at once would not fit the registers
          float s[32], d[32];
          const bool work = !idle && first + e < cols;
          if (work) {
            tc_ld32(lanes + first + e, reinterpret_cast<uint32_t*>(s));
            tc_ld32(lanes + G::DP + first + e, reinterpret_cast<uint32_t*>(d));
            tc_ld_wait();
            tc_loaded<32>(reinterpret_cast<uint32_t*>(s));
            tc_loaded<32>(reinterpret_cast<uint32_t*>(d));
          }
          if (e + 32 == HALF) {                       // the last columns are in registers: the next scores may come
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&hdr->s_free));
          }
          uint32_t pw[16], dw[16];
          if (work && !KEYS && !whole) {    // masked keys: p = 0 (the scale is positive here, see attention_tc_takes) and ds = 0
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (!(bits[e >> 5] >> k & 1u)) { s[k] = -AT_INF; d[k] = -nd; }
          }
          if (work) {
#pragma unroll
            for (int k = 0; k < 32; k += 4) {
              float4 l4, d4;
              if (KEYS) {
                l4 = *reinterpret_cast<const float4*>(st + e + k);
                d4 = *reinterpret_cast<const float4*>(st + CT + e + k);
              } else {
                l4 = make_float4(nl, nl, nl, nl); d4 = make_float4(nd, nd, nd, nd);
              }
#pragma unroll
              for (int z = 0; z < 2; ++z) {
                const int x = k + 2 * z;
                const float2 ex = fma2(make_float2(s[x], s[x + 1]), make_float2(c, c), z ? make_float2(l4.z, l4.w) : make_float2(l4.x, l4.y));
                float2 p = make_float2(ex2(ex.x), ex2(ex.y));
                float2 ds = mul2(p, add2(make_float2(d[x], d[x + 1]), z ? make_float2(d4.z, d4.w) : make_float2(d4.x, d4.y)));
                if (!KEYS) rest[z] = add2(rest[z], ds);
                pw[x >> 1] = KEYS && !row_ok ? 0u : pack_bf16(p.x, p.y);
                dw[x >> 1] = KEYS && !row_ok ? 0u : pack_bf16(ds.x, ds.y);
              }
            }
          }
          if (e == 0 && n > 0) {          // the previous P and dS have been read
            ok = at_wait(smem_u32(&hdr->mixed), (n - 1) & 1, abort_flag, status, 30, t.wait_limit);
            if (!ok) break;
            tc_fence_after();
          }
          if (work) {
            tc_st16(lanes + G::P + (first + e) / 2, pw);
            tc_st16(lanes + G::DS + (first + e) / 2, dw);
          }
        }
        if (!ok) break;
        if (!KEYS && !whole) {          // rows of K that must not be read; the scores are done with the tile
          const int k = lane + 32 * (warp & 3);         // four warps share the half's keys
          if (k < HALF) {
            uint32_t word = bits[0];
#pragma unroll
            for (int e = 1; e < HALF / 32; ++e) word = (k >> 5) == e ? bits[e] : word;
            if (!(word >> (k & 31) & 1u)) {
              unsigned char* p = smem_raw + (scol - raw) + slot * 2 * G::CTILE + (first + k) * 128;
#pragma unroll
              for (int e = 0; e < DC * 8; ++e) *reinterpret_cast<uint4*>(p + (e >> 3) * G::CBOX + (e & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
          }
          fence_async_smem();
        }
        tc_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&hdr->p_full));
        if (++slot == (uint32_t)G::NS) { slot = 0; sphase ^= 1u; }
      }
      if (!ok) break;
      // Results: dk by the first four warps and dv by the others, dq by halves of its channels, into the row tile's operand buffers (128-byte swizzle).
      constexpr int SPAN = KEYS ? DC * 64 : DC * 32;
      const int ch0 = KEYS ? 0 : half * SPAN;
      if (it.n == 0) {                 // no key in reach: zeros, and no buffer that is this row tile's
        const int rows = KEYS ? a.Lk : a.Lq, heads = KEYS ? a.Hkv : a.H, per = a.D / 8;
        for (int e = threadIdx.x; e < AT_M * per; e += EW_WARPS * 32) {
          const int z = it.row0 + e / per;
          const int64_t at = (((int64_t)it.b * rows + z) * heads + it.h) * a.D + e % per * 8;
          if (z < rows) {
            if (KEYS ? a.dk : a.dq) *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(KEYS ? a.dk : a.dq) + at) = make_uint4(0, 0, 0, 0);
            if (KEYS) *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.dv) + at) = make_uint4(0, 0, 0, 0);
          }
        }
        __syncwarp();
        continue;
      }
      ok = at_wait(smem_u32(&hdr->acc_full), turn.seq & 1, abort_flag, status, 31, t.wait_limit);
      if (!ok) break;
      tc_fence_after();
      const uint32_t from = KEYS ? (half ? G::ACC2 : G::ACC1) : G::ACC1 + half * SPAN;
      float corr = 0.f;
      if (!KEYS) {
        // Over a row ds sums to zero.  What it sums to is the error of delta, which comes from a result that was rounded, with weights that were rounded: it is taken out, times sum p k, here,
        // and out of delta itself for dk and dv.  The row's two threads join their columns' sums (in the room of the statistics, which this kernel has none of).
        float* joined = reinterpret_cast<float*>(smem_raw + (sstat - raw));
        static_assert(2 * AT_M <= G::NS * 2 * CT, "room for the sums");
        joined[half * AT_M + r] = (rest[0].x + rest[0].y) + (rest[1].x + rest[1].y);
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&hdr->summed));
        ok = at_wait(smem_u32(&hdr->summed), turn.seq & 1, abort_flag, status, 34, t.wait_limit);
        if (!ok) break;
        corr = joined[r] + joined[AT_M + r];
        if (half == 0 && row < a.Lq) g.nd_out[((int64_t)it.b * a.H + it.h) * g.pitch + row] = nd - corr;
        if (!a.dq) {                  // for delta alone
          tc_fence_before();
          __syncwarp();
          if (lane == 0) { mbar_arrive(smem_u32(&hdr->acc_free)); mbar_arrive(smem_u32(&hdr->staged[turn.buffer()])); }
          turn.next();
          continue;
        }
      }
      const float f = KEYS && half ? 1.f : it.end == 1 ? 0.f : a.scale;      // one key: its weight is one whatever its score
      unsigned char* stage = smem_raw + (srow - raw) + turn.buffer() * 2 * G::RTILE + (KEYS ? half * G::RTILE : 0) + r * 128;
      const bool zero = KEYS && !row_ok;
#pragma unroll 1
      for (int e = 0; e < SPAN; e += 32) {
        float v[32], m[KEYS ? 1 : 32];
        tc_ld32(lanes + from + e, reinterpret_cast<uint32_t*>(v));
        if (!KEYS) tc_ld32(lanes + from + e + (G::ACC2 - G::ACC1), reinterpret_cast<uint32_t*>(m));
        tc_ld_wait();
        tc_loaded<32>(reinterpret_cast<uint32_t*>(v));
        if (!KEYS) tc_loaded<KEYS ? 0 : 32>(reinterpret_cast<uint32_t*>(m));
        if (e + 32 == SPAN) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&hdr->acc_free));
        }
        if (!KEYS) {
#pragma unroll
          for (int k = 0; k < 32; ++k) v[k] = fmaf(-corr, m[KEYS ? 0 : k], v[k]);
        }
        const int ch = ch0 + e;
#pragma unroll
        for (int k = 0; k < 32; k += 8) {
          uint32_t w[4];
#pragma unroll
          for (int z = 0; z < 4; ++z) w[z] = zero ? 0u : pack_bf16(v[k + 2 * z] * f, v[k + 2 * z + 1] * f);
          *reinterpret_cast<uint4*>(stage + (ch >> 6) * G::RBOX + ((((ch & 63) + k) >> 3 ^ (r & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&hdr->staged[turn.buffer()]));
      turn.next();
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == SCORES) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

// -lse and -delta = -<dy, o> of every row, in rows of `pitch`: LANES lanes a row, 8 channels each.
template <int LANES>
__global__ void __launch_bounds__(256) attn_row_stats_kernel(const AttnArgs a, float* nl, float* nd, int pitch) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) / LANES;       // b, row, h: the heads of a row lie together
  const int lane = threadIdx.x % LANES;
  if (i >= (int64_t)a.B * pitch * a.H) return;
  const int h = (int)(i % a.H);
  const int64_t bl = i / a.H, b = bl / pitch;
  const int l = (int)(bl - b * pitch);
  float s = 0.f;
  if (l < a.Lq && lane * 8 < a.D) {
    const uint4 x = __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.o) + ((b * a.Lq + l) * a.H + h) * a.D) + lane);
    const uint4 y = __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.dy) + b * a.g_sb + l * a.g_sl + h * a.g_sh) + lane);
    const __nv_bfloat162 *u = reinterpret_cast<const __nv_bfloat162*>(&x), *v = reinterpret_cast<const __nv_bfloat162*>(&y);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 p = __bfloat1622float2(u[k]), q = __bfloat1622float2(v[k]);
      s = fmaf(p.x, q.x, s); s = fmaf(p.y, q.y, s);
    }
  }
  const uint32_t team = LANES == 32 ? 0xffffffffu : ((1u << LANES) - 1u) << (threadIdx.x % 32 / LANES * LANES);      // (the last warp's other rows may not be there)
  for (int w = LANES / 2; w > 0; w >>= 1) s += __shfl_xor_sync(team, s, w);
  if (lane == 0) {
    const int64_t at = (b * a.H + h) * pitch + l;
    nl[at] = l < a.Lq ? -__ldg(a.lse + (b * a.H + h) * a.Lq + l) : -AT_INF;
    nd[at] = -s;
  }
}

template <int DC, bool KEYS>
int launch(const AttnArgs& a, GradArgs g, cudaStream_t st) {
  using G = Grad<DC>;
  CUtensorMap tq, tk, tv, tg, t1, t2;
  const int q_rows = KEYS ? G::CT : AT_M, k_rows = KEYS ? AT_M : G::CT;
  int rc = fovi::encode_rows(&tq, &g.t.q, a.q, a.q_sb, a.q_sl, a.q_sh, a.B, a.Lq, a.H, a.D, q_rows);
  if (!rc) rc = fovi::encode_rows(&tg, &g.t.g, a.dy, a.g_sb, a.g_sl, a.g_sh, a.B, a.Lq, a.H, a.D, q_rows);
  if (!rc) rc = fovi::encode_rows(&tk, &g.t.k, a.k, a.k_sb, a.k_sl, a.k_sh, a.B, a.Lk, a.Hkv, a.D, k_rows);
  if (!rc) rc = fovi::encode_rows(&tv, &g.t.v, a.v, a.v_sb, a.v_sl, a.v_sh, a.B, a.Lk, a.Hkv, a.D, k_rows);
  const int64_t L = KEYS ? a.Lk : a.Lq, heads = KEYS ? a.Hkv : a.H;
  fovi::TcView whole;
  const void *q_like = a.dq ? a.dq : a.o, *k_like = a.dk ? a.dk : a.dv;        // (what is not wanted is not stored, but its map wants an address)
  if (!rc) rc = fovi::encode_rows(&t1, &whole, KEYS ? k_like : q_like, L * heads * a.D, heads * a.D, a.D, a.B, (int)L, (int)heads, a.D, AT_M);
  if (!rc) rc = fovi::encode_rows(&t2, &whole, KEYS ? a.dv : q_like, L * heads * a.D, heads * a.D, a.D, a.B, (int)L, (int)heads, a.D, AT_M);
  if (rc) return rc;
  g.tiles = ((KEYS ? a.Lk : a.Lq) + AT_M - 1) / AT_M;
  const int64_t items = (int64_t)g.tiles * (KEYS ? a.Hkv : a.H) * a.B;
  if (items > INT_MAX - 65536) return FOVI_ERR_UNSUPPORTED;
  g.items = (int)items;
  const int grid = std::min(g.items, fovi::sm_count());
  FOVI_CUDA(cudaFuncSetAttribute(attn_tc_grad_kernel<DC, KEYS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)G::SMEM));
  FOVI_CUDA(fovi::launch_pdl(attn_tc_grad_kernel<DC, KEYS>, grid, GR_THREADS, G::SMEM, st, tq, tk, tv, tg, t1, t2, g));
  return fovi::after_launch("attn_tc_grad_kernel");
}

}  // namespace

// Statistics of a row of queries: Lq rounded up to 16, as far as an MMA reads a last tile; copies of a whole tile may read up to 128 values more.
static int64_t stats_pitch(int Lq) { return ((int64_t)Lq + 15) / 16 * 16; }
int64_t fovi::attention_tc_backward_bytes(int B, int Lq, int H) { return (int64_t)B * H * stats_pitch(Lq) * 8 + 128 * 4; }

int fovi::launch_attention_tc_backward(const AttnArgs& a, void* work, cudaStream_t st, bool selftest) {
  GradArgs g = {};
  g.t.a = a;
  g.t.wait_limit = selftest ? 4096u : WAIT_LIMIT;
  g.t.skip_loads = selftest;
  int rc = attention_tc_status(&g.t.status);
  if (rc) return rc;
  g.pitch = (int)stats_pitch(a.Lq);
  const int64_t rows = (int64_t)a.B * a.H * g.pitch, blocks = (rows * (a.D <= 64 ? 8 : 16) + 255) / 256;
  if (blocks > INT_MAX) return FOVI_ERR_UNSUPPORTED;
  float* nl = static_cast<float*>(work);
  g.nl = nl; g.nd = g.nd_out = nl + rows;
  if (a.D <= 64) attn_row_stats_kernel<8><<<(int)blocks, 256, 0, st>>>(a, nl, nl + rows, g.pitch);
  else attn_row_stats_kernel<16><<<(int)blocks, 256, 0, st>>>(a, nl, nl + rows, g.pitch);
  rc = after_launch("attn_row_stats_kernel");
  // dq's kernel mends delta for dk too, so it also runs where dq is not wanted (then without its products and its result): dk is the same bits either way.  For dk and dv alone that costs
  // 772 us in place of 444 (257 queries over 1028 keys, 256 x 6 heads of 64 channels; with dq 800); dv does without.
  if (!rc && (a.dq || a.dk)) rc = a.D <= 64 ? launch<1, false>(a, g, st) : launch<2, false>(a, g, st);
  if (!rc && a.dv) rc = a.D <= 64 ? launch<1, true>(a, g, st) : launch<2, true>(a, g, st);
  return rc;
}
