// Matrix products of a token block on the tensor cores.
//
//   D[256 rows, ct columns] = sum over k of A[row, k] B[column, k]          bf16 with float32 sums, or 8-bit integers with 32-bit integer sums
//
// A cluster of two CTAs shares a tile (tcgen05.mma with cta_group::2, M = 256): each stages its 128 rows of A and half of B's ct rows, 128 bytes of k (64 bf16, 128 integers) a stage,
// by tensor copies.  An operand whose k is contiguous is K-major; one that lies the other way round (weights in the input gradients, both operands of a weight gradient) is read MN-major,
// as 64-column boxes, so nothing is transposed in memory.  Two accumulators in tensor memory: a tile's epilogue runs under the next one's products.
// Persistent: of n pairs each takes every n-th tile.  Roles: warps 0-7 epilogue (a row per thread, the two halves take turns on 32-column chunks), warp 8 MMAs (of the pair's first CTA), warp 9 copies.
// All waits are bounded.
//
// What becomes of a tile:
//   GATED    accumulator columns of the first half are g, of the second u, since the first CTA stages rows of Wg and the second the same rows of Wu: h = act(g) u
//   GRAD     the tile is dh; g and u are read, dg and du written
//            Both move 8 and 10 bytes a hidden value, which is what bounds them where C is small, so their tiles go through shared memory as tensor copies, 32 rows x 32 columns of a warp at
//            a time: with a row per thread in global memory every instruction touched 32 lines, and the load/store unit bound them (65792 x 384 x 1024: 227 and 293 us, now 124 and 132:
//            5.4 TB/s of theirs).
//   STORE    bf16 result with a bias, or with k in parts a float32 part, joined by a second kernel in their order
//   SCALED   integer sums times the scales
// Where C is large the power limit bounds it: 16448 tokens, 1280 x 5120 channels, projections 1.30 PFLOP/s, down 1.32, input gradients 1.26, weight gradients 1.36 (from 1.2 to 1.3 sustained
// for library products of these sizes), hidden gradients 0.95, whose tiles' arithmetic is longer than their products.  8-bit 16448 x 1280 -> 5120 in 86 to 97 us, 2.2 to 2.5 P a
// second: bound by the epilogue's stores, a row a thread in pieces of 32 bytes, 32 lines an instruction (62 us without them, 512 clocks a stage of 256 columns).
#include <algorithm>

#include "product_pair.cuh"
#include "product_split.cuh"
#include "product_tc.cuh"

using fovi::Hidden;
using fovi::TcMatrix;
using fovi::TcShape;
using fovi::TcTask;

namespace {

__device__ int g_status;           // wait site at which a kernel gave up, see fovi_product_check: one word per device

enum { GATED = 0, GRAD = 1, STORE = 2, SCALED = 3 };
constexpr int EPI_WARPS = 8, PT_THREADS = (EPI_WARPS + 2) * 32;
constexpr uint32_t A_BYTES = 16384, STAGE_BYTES = 2 * A_BYTES;      // a CTA's 128 rows of A and up to 128 rows of B
constexpr int MOST_STAGES = 5, GROUPS = 3;
// Shared memory of an epilogue warp.  GATED: a chunk's g and u (high 4 KB, low 2 KB) and h (2 KB) on their way out.  GRAD: two such places for g and u on their way in, dg and du go out from
// over the high parts.  Otherwise: 32 rows x 32 columns (odd pitch), or 64 factors and biases.
template <int EPI> struct Sizes {
  static constexpr uint32_t SCRATCH = EPI == GATED ? 8192 : EPI == GRAD ? 12288 : 32 * 33 * 4;
  static constexpr int STAGES = EPI == GATED ? 5 : EPI == GRAD ? 4 : 5;
  static constexpr uint32_t SMEM = 1024 + 1024 + EPI_WARPS * SCRATCH + STAGES * STAGE_BYTES;
  static_assert(SMEM <= 227 * 1024 && SCRATCH * EPI_WARPS % 1024 == 0, "");
};

struct PtMaps { CUtensorMap a[GROUPS], b[GROUPS], high, low, out[2]; };       // a, b: of each task, or of each segment of k; out: h, or dg and du

struct PtArgs {
  int tasks, first[GROUPS + 1];            // tiles first[t] .. first[t + 1] - 1 belong to task t
  int n_mt[GROUPS], n_nt[GROUPS], m[GROUPS], n[GROUPS];
  void* y[GROUPS];
  int64_t part[GROUPS];                    // parts of k: where a task's begin in `work` (float32)
  int kb0, kb, splits;                     // stages of the first segment of k, of all, parts
  int ct;
  const void *bias, *bias2;
  Hidden hidden; float* sums;
  const float *scale, *wscale, *bias_f; int y_f32;
  float* work;
  int* status; uint32_t wait_limit; int skip_loads;
};

struct PtHeader {
  uint64_t full[MOST_STAGES], empty[MOST_STAGES], acc_full[2], acc_empty[2], drain, came[EPI_WARPS][2];
  uint32_t tmem_base;
  int abort_flag;
};

// Copies of a warp's chunk, issued by one lane.
__device__ __forceinline__ void pt_load_own(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
               ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void pt_store(const CUtensorMap* map, uint32_t src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map), "r"(src), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }      // this thread's stores have read shared memory
__device__ __forceinline__ void bulk_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void async_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void put16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void get16(uint32_t at, uint32_t* w) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ uint32_t get4(uint32_t at) {
  uint32_t w;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(at) : "memory");
  return w;
}
// Place of 16-byte piece c of row r in a tile of 128-byte or 64-byte rows, swizzled over that many bytes: eight rows' pieces lie in eight bank groups.
__device__ __forceinline__ uint32_t at128(int r, int c) { return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4)); }
__device__ __forceinline__ uint32_t at64(int r, int c) { return (uint32_t)(r * 64 + ((c ^ (r >> 1 & 3)) << 4)); }
// The larger of two, not a number where one is not.
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// act(g) and act'(g) of two values, to a few units of float32: what is rounded to bf16 behind them.  The logistic function takes an exponential each and one reciprocal for both,
// 1/a = b/(ab), since those units are what bounds a tile's arithmetic.  Exponents are cut at 2^60, so that the product stays finite, and the factor g with them, at -60 ln 2: from there on
// value and slope stand still, at -4e-17.  In the slope p + a (1 - p) the last factor is exp(-g) p: from p itself it would be its error, 2^-23, which a gate of 1e5 and more makes
// a slope of.  The exponent's cut drops what is not a number, as the pair shares its reciprocal; the factor's keeps it.
template <int ACT> __device__ __forceinline__ float2 act_pair(float2 g, float2* slope) {
  if (ACT == fovi::ACT_SILU) {
    const float2 x = mul2(g, both(-1.4426950408889634f));
    float2 q;
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(q.x) : "f"(fminf(x.x, 60.f)));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(q.y) : "f"(fminf(x.y, 60.f)));
    const float2 e = add2(q, both(1.f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(e.x * e.y));
    const float2 p = mul2(both(r), make_float2(e.y, e.x)), a = mul2(make_float2(max_nan(g.x, -41.588831f), max_nan(g.y, -41.588831f)), p);
    if (slope) *slope = fma2(a, mul2(q, p), p);
    return a;
  }
  const float2 x = mul2(g, both(0.70710678118654752f));
  const float2 p = fma2(make_float2(erff(x.x), erff(x.y)), both(0.5f), both(0.5f));
  if (slope) {
    const float2 q = mul2(mul2(g, both(-0.5f)), g);
    *slope = fma2(mul2(g, both(0.39894228040143268f)), make_float2(__expf(q.x), __expf(q.y)), p);
  }
  return mul2(g, p);
}

// A value whose upper 24 bits are it, rounded: infinity and not-a-number stay what they are, and finite values from the largest of 24 bits on (0x1.fffep127) finite.
__device__ __forceinline__ uint32_t upper24(uint32_t v) { return fabsf(__uint_as_float(v)) < 0x1.fffep127f ? v + 0x80u : v; }

// Sums of 32 columns over the lanes, a column at a time: column c's value of every lane goes in, and after the last the sum of column `lane` comes out.  Two neighbours' sums are halved at
// each level: a lane keeps the one whose number has its bit.  31 exchanges in all, in a fixed order.
struct ColumnSums {
  float level[5];
  __device__ __forceinline__ float join(float a, float b, int bit, int lane) {
    const bool upper = lane & bit;
    return (upper ? b : a) + __shfl_xor_sync(0xffffffffu, upper ? a : b, bit);
  }
  __device__ __forceinline__ float add(int c, float v, int lane) {           // c: a constant
#pragma unroll
    for (int l = 0; l < 5; ++l) {
      if (!(c >> l & 1)) { level[l] = v; return v; }
      v = join(level[l], v, 1 << l, lane);
    }
    return v;
  }
};

struct Tile { int task, mt, nt, k0, k1, split; };
__device__ __forceinline__ Tile tile_of(const PtArgs& a, int item) {
  Tile t;
  t.task = 0;
  if (a.tasks > 1) t.task = item >= a.first[2] ? 2 : item >= a.first[1] ? 1 : 0;
  int r = item - a.first[t.task];
  t.nt = r % a.n_nt[t.task];
  r /= a.n_nt[t.task];
  t.mt = r % a.n_mt[t.task];
  t.split = r / a.n_mt[t.task];
  t.k0 = (int)((int64_t)a.kb * t.split / a.splits);
  t.k1 = (int)((int64_t)a.kb * (t.split + 1) / a.splits);
  return t;
}

// 32 columns of a row tile of 32 rows (a row per lane) into [m, n] with no alignment: through the warp's scratch, so that lanes write neighbouring columns.
template <typename T> __device__ __forceinline__ void store_any(T* y, int64_t n, int64_t row0, int64_t m, int c0, const float* v, float* scratch, int lane) {
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 32; ++i) scratch[lane * 33 + i] = v[i];
  __syncwarp();
  if (c0 + lane < n) {
    const int rows = (int)min((int64_t)32, m - row0);
    T* to = y + row0 * n + c0 + lane;
#pragma unroll 8
    for (int r = 0; r < rows; ++r) to[r * n] = from_float<T>(scratch[r * 33 + lane]);
  }
  __syncwarp();
}

template <int EPI, bool A_MN, bool B_MN, bool I8, int ACT, bool WHOLE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PT_THREADS, 1) product_tc_kernel(const __grid_constant__ PtMaps maps, const __grid_constant__ PtArgs a) {
  extern __shared__ unsigned char smem_raw[];
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  PtHeader* hdr = reinterpret_cast<PtHeader*>(smem_raw + (base - raw));
  constexpr uint32_t SCRATCH = Sizes<EPI>::SCRATCH;
  constexpr int STAGES = Sizes<EPI>::STAGES;
  const uint32_t stages0 = base + 1024u + EPI_WARPS * SCRATCH;
  volatile int* abort_flag = &hdr->abort_flag;
  const int warp = warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int rank = (int)pt_rank(), worker = blockIdx.x >> 1, workers = gridDim.x >> 1;
  const int half = a.ct / 2, total = a.first[a.tasks];
  constexpr int KS = I8 ? 128 : 64;               // values of k a stage

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(smem_u32(&hdr->full[s]), 1); mbar_init(smem_u32(&hdr->empty[s]), 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(smem_u32(&hdr->acc_full[i]), 1); mbar_init(smem_u32(&hdr->acc_empty[i]), 2 * EPI_WARPS); }
    mbar_init(smem_u32(&hdr->drain), 1);
    if (EPI == GRAD)
      for (int i = 0; i < 2 * EPI_WARPS; ++i) mbar_init(smem_u32(&hdr->came[0][0]) + 8 * i, 1);
    hdr->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == EPI_WARPS) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&hdr->tmem_base)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  tc_fence_before();
  pt_sync();
  tc_fence_after();
  const uint32_t tmem = hdr->tmem_base;

  if (warp == EPI_WARPS + 1) {
    // ------------------------------------------------------------ copies
    const uint32_t b_bytes = B_MN ? (uint32_t)((half + 63) / 64) * 8192u : (uint32_t)half * 128u;
    uint32_t s = 0, ph = 0;
    bool ok = !a.skip_loads;
    for (int item = worker; item < total && ok; item += workers) {
      const Tile t = tile_of(a, item);
      const int m0 = t.mt * 256 + rank * 128, n0 = EPI == GATED ? t.nt * half : t.nt * a.ct + rank * half;
      for (int kb = t.k0; kb < t.k1; ++kb) {
        ok = mbar_wait_warp(smem_u32(&hdr->empty[s]), ph ^ 1u, abort_flag, a.status, 41, a.wait_limit);
        if (!ok) break;
        const int seg = kb >= a.kb0 ? 1 : 0, k = (kb - (seg ? a.kb0 : 0)) * KS;
        const CUtensorMap *ma = &maps.a[t.task + seg], *mb = &maps.b[EPI == GATED ? rank : t.task + seg];
        const uint32_t full = pt_map(smem_u32(&hdr->full[s]), 0), sa = stages0 + s * STAGE_BYTES, sb = sa + A_BYTES;
        if (elect_one()) {
          if (rank == 0) mbar_expect_tx(smem_u32(&hdr->full[s]), 2u * (A_BYTES + b_bytes));      // of both CTAs
          if (A_MN) {
            pt_load(sa, ma, full, m0, k);
            pt_load(sa + 8192u, ma, full, m0 + 64, k);
          } else {
            pt_load(sa, ma, full, k, m0);
          }
          if (B_MN) {
            for (int j = 0; j < half; j += 64) pt_load(sb + j * 128u, mb, full, n0 + j, k);
          } else {
            pt_load(sb, mb, full, k, n0);
          }
        }
        __syncwarp();
        if (++s == STAGES) { s = 0; ph ^= 1u; }
      }
    }
    if (lane == 0 && *abort_flag) {
      for (int i = 0; i < 64; ++i) __nanosleep(1000);    // copies in flight land before this CTA's shared memory goes away
    }
  } else if (warp == EPI_WARPS) {
    // ------------------------------------------------------------ products (see elect_one)
    if (rank == 0) {
      const uint32_t idesc = (I8 ? 2u << 4 : 1u << 4) | (1u << 7) | (1u << 10) | (A_MN ? 1u << 15 : 0u) | (B_MN ? 1u << 16 : 0u) | ((uint32_t)(a.ct >> 3) << 17) | (16u << 24);
      const uint64_t desc_a = smem_desc(0, A_MN ? 8192u : 16u, 1024u, 2u), desc_b = smem_desc(0, B_MN ? 8192u : 16u, 1024u, 2u);
      const uint32_t u_stages0 = warp_uniform(stages0), u_tmem = warp_uniform(tmem);
      uint32_t s = 0, ph = 0, acc = 0, aph = 0;
      bool ok = true;
      for (int item = worker; item < total && ok; item += workers) {
        const Tile t = tile_of(a, item);
        const int steps = warp_uniform(t.k1 - t.k0);
        ok = mbar_wait_warp(smem_u32(&hdr->acc_empty[acc]), aph ^ 1u, abort_flag, a.status, 42, a.wait_limit);
        if (!ok) break;
        tc_fence_after();
        const uint32_t d = u_tmem + acc * 256u;
        for (int st = 0; st < steps; ++st) {
          ok = mbar_wait_warp(smem_u32(&hdr->full[s]), ph, abort_flag, a.status, 43, a.wait_limit);
          if (!ok) break;
          tc_fence_after();
          const uint32_t sa = u_stages0 + s * STAGE_BYTES;
          const uint64_t da = desc_a + (sa >> 4), db = desc_b + ((sa + A_BYTES) >> 4);
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) pt_mma<I8>(d, da + kk * (A_MN ? 128u : 2u), db + kk * (B_MN ? 128u : 2u), idesc, (st | kk) ? 1u : 0u);
            pt_commit(smem_u32(&hdr->empty[s]));
            if (st == steps - 1) pt_commit(smem_u32(&hdr->acc_full[acc]));
          }
          __syncwarp();
          if (++s == STAGES) { s = 0; ph ^= 1u; }
        }
        if (!ok) break;
        if (++acc == 2) { acc = 0; aph ^= 1u; }
      }
      if (*abort_flag && elect_one()) {
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(&hdr->drain)) : "memory");
        for (uint32_t i = 0; i < (1u << 20); ++i)
          if (mbar_try_wait(smem_u32(&hdr->drain), 0)) break;
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int quarter = warp & 3, turn = warp >> 2;
    float* scratch = reinterpret_cast<float*>(smem_raw + (base - raw) + 1024u + warp * SCRATCH);
    const uint32_t place = base + 1024u + warp * SCRATCH;
    const int width = EPI == GATED ? half : a.ct;                     // columns of a tile; this warp's chunks of 32 are turn, turn + 2, ...
    auto chunks_of = [&](const Tile& t) {                             // columns from the end on are not written
      const int end = EPI == GATED || EPI == GRAD ? (int)a.hidden.pitch : a.n[t.task];
      return min(width / 32, (end - t.nt * width + 31) / 32);
    };
    auto row_of = [&](const Tile& t) { return t.mt * 256 + rank * 128 + quarter * 32; };
    uint32_t acc = 0, aph = 0;
    // GRAD: g and u of this warp's chunks, two on their way.  The next to be asked for is chunk next_c of next_item.
    int next_item = worker, next_c = turn, next_chunks = 0, next_col = 0, next_row = 0, asked = 0, taken = 0;
    auto next_tile = [&]() {                         // on to a tile with a chunk for this warp
      for (next_c = turn; next_item < total; next_item += workers) {
        const Tile t = tile_of(a, next_item);
        next_chunks = chunks_of(t);
        next_col = t.nt * width;
        next_row = row_of(t);
        if (turn < next_chunks) return;
      }
    };
    auto ask = [&]() {
      if (next_item >= total) return;
      if (lane == 0) {
        const uint32_t to = place + (asked & 1) * 6144u, bar = smem_u32(&hdr->came[warp][asked & 1]);
        mbar_expect_tx(bar, 6144u);
        pt_load_own(to, &maps.high, bar, 2 * (next_col + 32 * next_c), next_row);
        pt_load_own(to + 4096u, &maps.low, bar, 2 * (next_col + 32 * next_c), next_row);
      }
      ++asked;
      next_c += 2;
      if (next_c >= next_chunks) { next_item += workers; next_tile(); }
    };
    if (EPI == GRAD) next_tile();
    if (EPI == GRAD && !a.skip_loads) { ask(); ask(); }
    for (int item = worker; item < total; item += workers) {
      const Tile t = tile_of(a, item);
      const int row0 = row_of(t), row = row0 + lane;
      const uint32_t t_base = tmem + ((uint32_t)(quarter * 32) << 16) + acc * 256u;
      const int M = a.m[t.task], N = a.n[t.task];
      const bool here = row < M;
      const int col0 = t.nt * width, chunks = chunks_of(t);
      float rs = 0.f, f0[4], f1[4];                   // asked for in front of the wait: the row's scale, and a column a lane of factors and biases for each of up to four chunks
      if (EPI == SCALED) rs = here ? __ldg(a.scale + row) : 0.f;
#pragma unroll
      for (int i = 0; i < (EPI == GATED ? 2 : 4); ++i) {
        const int n = col0 + 32 * (turn + 2 * i) + lane;
        const bool in = turn + 2 * i < chunks && n < N;
        const __nv_bfloat16 *b0 = static_cast<const __nv_bfloat16*>(a.bias), *b1 = static_cast<const __nv_bfloat16*>(a.bias2);
        f0[i] = f1[i] = 0.f;
        if (EPI == SCALED) {
          if (in) f0[i] = __ldg(a.wscale + n);
          if (in && a.bias_f) f1[i] = __ldg(a.bias_f + n);
        } else if (EPI == GATED || (EPI == STORE && a.splits == 1)) {
          if (in && b0) f0[i] = __bfloat162float(__ldg(b0 + n));
          if (EPI == GATED && in && b1) f1[i] = __bfloat162float(__ldg(b1 + n));
        }
      }
      if (!mbar_wait_warp(smem_u32(&hdr->acc_full[acc]), aph, abort_flag, a.status, 44, a.wait_limit)) break;
      tc_fence_after();
      // This warp has read the accumulator.  The arrival hands over tensor memory alone: the wait for the loads has put their values into registers, and the fences on both sides order the next products behind it.
      // So it is relaxed: a release would also wait for the warp's stores to arrive in memory, which nobody behind this barrier reads.
      auto release = [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(pt_map(smem_u32(&hdr->acc_empty[acc]), 0)) : "memory");
      };
      if (turn >= chunks) release();
      bool lost = false;
#pragma unroll
      for (int ci = 0; ci < (EPI == GATED ? 2 : 4); ++ci) {
        const int c = turn + 2 * ci, c0 = col0 + 32 * c;
        if (c >= chunks) break;
        if (EPI == GATED) {
          uint32_t g[32], u[32];
          tc_ld32(t_base + 32 * c, g);
          tc_ld32(t_base + half + 32 * c, u);
          tc_ld_wait();
          pt_loaded(g);
          pt_loaded(u);
          if (c + 2 >= chunks) release();
          if (a.bias) {
#pragma unroll
            for (int i = 0; i < 32; ++i) g[i] = __float_as_uint(__uint_as_float(g[i]) + __shfl_sync(0xffffffffu, f0[ci], i));
          }
          if (a.bias2) {
#pragma unroll
            for (int i = 0; i < 32; ++i) u[i] = __float_as_uint(__uint_as_float(u[i]) + __shfl_sync(0xffffffffu, f1[ci], i));
          }
          if (lane == 0) bulk_read();                 // the chunk before has left this place
          __syncwarp();
          if (a.hidden.high) {
#pragma unroll
            for (int m = 0; m < 2; ++m) {
              uint32_t v[32];
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = upper24(m ? u[i] : g[i]);
#pragma unroll
              for (int i = 0; i < 4; ++i)
                put16(place + at128(lane, 4 * m + i), __byte_perm(v[8 * i], v[8 * i + 1], 0x7632), __byte_perm(v[8 * i + 2], v[8 * i + 3], 0x7632),
                      __byte_perm(v[8 * i + 4], v[8 * i + 5], 0x7632), __byte_perm(v[8 * i + 6], v[8 * i + 7], 0x7632));
              uint32_t lo[8];
#pragma unroll
              for (int i = 0; i < 8; ++i)
                lo[i] = __byte_perm(__byte_perm(v[4 * i], v[4 * i + 1], 0x0051), __byte_perm(v[4 * i + 2], v[4 * i + 3], 0x0051), 0x5410);
#pragma unroll
              for (int i = 0; i < 2; ++i) put16(place + 4096u + at64(lane, 2 * m + i), lo[4 * i], lo[4 * i + 1], lo[4 * i + 2], lo[4 * i + 3]);
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t h[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int e = 8 * i + 2 * j;
              const float2 v = mul2(act_pair<ACT>(make_float2(__uint_as_float(g[e]), __uint_as_float(g[e + 1])), nullptr),
                                    make_float2(__uint_as_float(u[e]), __uint_as_float(u[e + 1])));
              h[j] = bf16_pair(v.x, v.y);
            }
            put16(place + 6144u + at64(lane, i), h[0], h[1], h[2], h[3]);
          }
          async_fence();
          __syncwarp();
          if (lane == 0) {                            // rows behind the last token are outside the tensors, and left out
            if (a.hidden.high) {
              pt_store(&maps.high, place, 2 * c0, row0);
              pt_store(&maps.low, place + 4096u, 2 * c0, row0);
            }
            pt_store(&maps.out[0], place + 6144u, c0, row0);
            bulk_commit();
          }
        } else if (EPI == GRAD) {
          const uint32_t from = place + (taken & 1) * 6144u;
          if (!mbar_wait_warp(smem_u32(&hdr->came[warp][taken & 1]), taken >> 1 & 1, abort_flag, a.status, 45, a.wait_limit)) { lost = true; break; }
          ++taken;
          uint32_t r[32], gu[32], lo[16];             // gu: g of 32 columns, then u
          tc_ld32(t_base + 32 * c, r);
#pragma unroll
          for (int i = 0; i < 8; ++i) get16(from + at128(lane, i), gu + 4 * i);
#pragma unroll
          for (int i = 0; i < 4; ++i) get16(from + 4096u + at64(lane, i), lo + 4 * i);
          tc_ld_wait();
          pt_loaded(r);
          if (c + 2 >= chunks) release();
          uint32_t dg[16], du[16];
          ColumnSums of_dg, of_du;
          float sum_g = 0.f, sum_u = 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float g[2], u[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int e = 2 * i + j;
              const uint32_t pick = (j ? 0x3244u : 0x1044u) + ((uint32_t)(e & 3) << 4);      // [two high bytes, low byte, any]
              g[j] = __uint_as_float(__byte_perm(gu[i], lo[e / 4], pick) & 0xffffff00u);
              u[j] = __uint_as_float(__byte_perm(gu[16 + i], lo[8 + e / 4], pick) & 0xffffff00u);
            }
            float2 d;
            const float2 dh = make_float2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), v = mul2(dh, act_pair<ACT>(make_float2(g[0], g[1]), &d));
            d = mul2(mul2(dh, make_float2(u[0], u[1])), d);
            dg[i] = bf16_pair(d.x, d.y);
            du[i] = bf16_pair(v.x, v.y);
            if (WHOLE) {
              of_dg.add(2 * i, d.x, lane); sum_g = of_dg.add(2 * i + 1, d.y, lane);
              of_du.add(2 * i, v.x, lane); sum_u = of_du.add(2 * i + 1, v.y, lane);
            }
          }
          __syncwarp();                               // every lane has its g and u
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            put16(from + at64(lane, i), dg[4 * i], dg[4 * i + 1], dg[4 * i + 2], dg[4 * i + 3]);
            put16(from + 2048u + at64(lane, i), du[4 * i], du[4 * i + 1], du[4 * i + 2], du[4 * i + 3]);
          }
          async_fence();
          __syncwarp();
          if (lane == 0) {
            pt_store(&maps.out[0], from, c0, row0);
            pt_store(&maps.out[1], from + 2048u, c0, row0);
            bulk_commit();
          }
          if (a.sums) {                               // of this warp's 32 rows; rows behind the last token are zeros of dy, and so of dg and du
            float* to = a.sums + (int64_t)(row0 >> 5) * 2 * a.hidden.pitch + c0;
            if (WHOLE) {                              // before they were rounded
              to[lane] = sum_g;
              to[a.hidden.pitch + lane] = sum_u;
            } else {                                  // of the rounded values, two columns a lane
              float2 sum = both(0.f);
              const uint32_t mine = from + (lane >> 4) * 2048u;
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                const uint32_t w = get4(mine + at64(i, lane >> 2 & 3) + (lane & 3) * 4u);
                sum = add2(sum, make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)));
              }
              *reinterpret_cast<float2*>(to + (lane >> 4) * a.hidden.pitch + 2 * (lane & 15)) = sum;
            }
          }
          if (lane == 0) bulk_read();
          __syncwarp();
          ask();
        } else {
          uint32_t r[32];
          float v[32];
          __syncwarp();
          scratch[lane] = f0[ci];
          if (EPI == SCALED) scratch[32 + lane] = f1[ci];
          __syncwarp();
          tc_ld32(t_base + 32 * c, r);
          tc_ld_wait();
          pt_loaded(r);
          if (c + 2 >= chunks) release();
          if (EPI == STORE && a.splits > 1) {
            if (here) {
              const int64_t pitch = (N + 31) / 32 * 32;
              float* to = a.work + a.part[t.task] + ((int64_t)t.split * M + row) * pitch + c0;
#pragma unroll
              for (int i = 0; i < 32; i += 8) st_global_32f(to + i, r + i);
            }
            continue;
          }
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = EPI == SCALED ? fmaf((float)(int)r[i] * rs, scratch[i], scratch[32 + i]) : __uint_as_float(r[i]) + scratch[i];
          void* y = a.y[t.task];
          const bool f32 = EPI == SCALED && a.y_f32;
          if (f32 && N % 8 == 0) {
            if (here) {
              float* to = static_cast<float*>(y) + (int64_t)row * N + c0;
#pragma unroll
              for (int i = 0; i < 32; i += 8) {
                uint32_t w[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] = __float_as_uint(v[i + j]);
                if (c0 + i < N) st_global_32(to + i, w);
              }
            }
          } else if (!f32 && N % 16 == 0) {
            if (here) {
              uint16_t* to = static_cast<uint16_t*>(y) + (int64_t)row * N + c0;
#pragma unroll
              for (int i = 0; i < 32; i += 16) {
                uint32_t w[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] = bf16_pair(v[i + 2 * j], v[i + 2 * j + 1]);
                if (c0 + i < N) st_global_32(to + i, w);
              }
            }
          } else if (f32) {
            store_any(static_cast<float*>(y), N, row0, M, c0, v, scratch, lane);
          } else {
            store_any(static_cast<__nv_bfloat16*>(y), N, row0, M, c0, v, scratch, lane);
          }
        }
      }
      if (lost) break;
      if (++acc == 2) { acc = 0; aph ^= 1u; }
    }
    if ((EPI == GATED || EPI == GRAD) && lane == 0) bulk_done();
    if (EPI == GRAD && *abort_flag && lane == 0) {
      for (int i = 0; i < 64; ++i) __nanosleep(1000);    // copies in flight, as above
    }
  }
  tc_fence_before();
  pt_sync();
  if (warp == EPI_WARPS) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// The parts of the products' k, added in their order, with the bias.  A thread for four columns; y counts the products.
struct JoinArgs { const float* part[GROUPS]; __nv_bfloat16* y[GROUPS]; int64_t m[GROUPS]; int n[GROUPS], splits; const __nv_bfloat16* bias; };
__global__ void __launch_bounds__(256) product_join_kernel(const __grid_constant__ JoinArgs a) {
  const int t = blockIdx.y, n = a.n[t];
  const uint32_t pitch = (n + 31) / 32 * 32, per = pitch / 4;
  const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t m = a.m[t], row = i >> 32 ? i / per : (uint32_t)i / per;
  const int c = (int)(i - row * per) * 4;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (row >= m || c >= n) return;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  const float* from = a.part[t] + row * pitch + c;
#pragma unroll 4
  for (int p = 0; p < a.splits; ++p) {
    float4 v;
    asm volatile("ld.global.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(from + p * m * pitch) : "memory");
    s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
  }
  float b[4] = {s.x, s.y, s.z, s.w};
  if (a.bias) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c + e < n) b[e] += __bfloat162float(__ldg(a.bias + c + e));
  }
  __nv_bfloat16* to = a.y[t] + row * n + c;
  if (n % 4 == 0) {
    *reinterpret_cast<uint2*>(to) = make_uint2(bf16_pair(b[0], b[1]), bf16_pair(b[2], b[3]));
  } else {
    for (int e = 0; e < 4 && c + e < n; ++e) to[e] = __float2bfloat16_rn(b[e]);
  }
}

// ------------------------------------------------------------------------------------------------------------ host
int pairs() { return std::max(1, fovi::sm_count() / 2); }

cudaError_t status_word(int** word) {
  static std::atomic<int*> known[64];
  return word_of(word, g_status, known);
}

// The cut with the least time by a count of clocks: 2 clocks a column and stage, about 1500 for a tile's start and end, and for k in parts their way through memory.
// `columns` of a tile are divided among `share` matrices (GATED: 2).
TcShape shape_of(const int64_t* m, const int* n, int tasks, int64_t kb, int share, bool may_split) {
  TcShape best{256, 1};
  double least = 1e300;
  const int64_t at_once = pairs();
  for (int ct = 256; ct >= 64; ct -= 64) {
    int64_t tiles = 0, values = 0;
    for (int t = 0; t < tasks; ++t) {
      tiles += (m[t] + 255) / 256 * ((n[t] * (int64_t)share + ct - 1) / ct);
      values += m[t] * ((n[t] + 31) / 32 * 32);
    }
    for (int s = 1; s <= (may_split ? 32 : 1) && (s == 1 || kb / s >= 4); ++s) {
      const double ways = s > 1 ? 5000 + (double)values * s * 8 / 3400 : 0;
      if (ways >= least) break;
      const double clocks = ways + (double)((tiles * s + at_once - 1) / at_once) * ((double)((kb + s - 1) / s) * std::max(2 * ct, 200) + 1500);
      if (clocks < least) { least = clocks; best = {ct, s}; }
    }
  }
  return best;
}

int map_k(CUtensorMap* m, const TcMatrix& x, bool bytes, int rows) {
  return fovi::encode_2d(m, x.p, bytes, (uint64_t)x.cols, (uint64_t)x.rows, (uint64_t)x.pitch * (bytes ? 1 : 2), bytes ? 128 : 64, (uint32_t)rows);
}
int map_mn(CUtensorMap* m, const TcMatrix& x) { return fovi::encode_2d(m, x.p, false, (uint64_t)x.cols, (uint64_t)x.rows, (uint64_t)x.pitch * 2, 64, 64); }

template <int EPI, bool A_MN, bool B_MN, bool I8, int ACT = 0, bool WHOLE = false> int launch(const PtMaps& maps, PtArgs& a, bool selftest, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  FOVI_CUDA(status_word(&a.status));
  a.wait_limit = selftest ? 4096u : WAIT_LIMIT;
  a.skip_loads = selftest;
  const int grid = 2 * std::min(a.first[a.tasks], pairs());
  auto kernel = product_tc_kernel<EPI, A_MN, B_MN, I8, ACT, WHOLE>;
  FOVI_CUDA(allow_shared(kernel, (int)Sizes<EPI>::SMEM, done));
  FOVI_CUDA(fovi::launch_pdl(kernel, grid, PT_THREADS, Sizes<EPI>::SMEM, st, maps, a));
  return fovi::after_launch("product_tc_kernel");
}

// Tensors of a row of hidden values a token, as boxes of 32 rows x 32 columns (high, low: of g and u side by side).
int map_hidden(PtMaps& maps, const Hidden& h, int64_t m) {
  if (!h.high) return FOVI_OK;
  const int rc = fovi::encode_2d(&maps.high, h.high, false, 2 * h.pitch, m, 4 * h.pitch, 64, 32);
  return rc ? rc : fovi::encode_2d(&maps.low, h.low, true, 2 * h.pitch, m, 2 * h.pitch, 64, 32, true);
}
int map_out(CUtensorMap* map, const void* p, int64_t pitch, int64_t m) { return fovi::encode_2d(map, p, false, pitch, m, 2 * pitch, 32, 32, true); }

// Tiles of each task, in order.
int tiles_of(PtArgs& a, int share) {
  int64_t at = 0;
  for (int t = 0; t < a.tasks; ++t) {
    a.first[t] = (int)at;
    a.n_mt[t] = (a.m[t] + 255) / 256;
    a.n_nt[t] = (int)(((int64_t)a.n[t] * share + a.ct - 1) / a.ct);
    at += (int64_t)a.n_mt[t] * a.n_nt[t] * a.splits;
  }
  if (at >= (1ll << 31) - (1 << 16)) return FOVI_ERR_UNSUPPORTED;
  for (int t = a.tasks; t <= GROUPS; ++t) a.first[t] = (int)at;
  return FOVI_OK;
}

int join(const PtArgs& a, cudaStream_t st) {
  JoinArgs j{};
  int64_t threads = 0;
  j.splits = a.splits;
  j.bias = static_cast<const __nv_bfloat16*>(a.bias);
  for (int t = 0; t < a.tasks; ++t) {
    j.part[t] = a.work + a.part[t]; j.y[t] = static_cast<__nv_bfloat16*>(a.y[t]); j.m[t] = a.m[t]; j.n[t] = a.n[t];
    threads = std::max(threads, (int64_t)a.m[t] * ((a.n[t] + 31) / 32 * 8));
  }
  FOVI_CUDA(fovi::launch_pdl(product_join_kernel, dim3((unsigned)((threads + 255) / 256), a.tasks), 256, 0, st, j));
  return fovi::after_launch("product_join_kernel");
}

int64_t stages_of(int64_t k) { return (k + 63) / 64; }

}  // namespace

int fovi::tc_gated(const TcMatrix& x, const TcMatrix& wg, const TcMatrix& wu, const void* bg, const void* bu, int act, const Hidden& to, cudaStream_t st) {
  PtArgs a{};
  PtMaps maps{};
  const int64_t m = x.rows;
  const int n = (int)wg.rows;
  a.tasks = 1; a.m[0] = (int)m; a.n[0] = n;
  a.kb0 = a.kb = (int)stages_of(x.cols);
  a.splits = 1;
  a.ct = shape_of(&m, &n, 1, a.kb, 2, false).ct;
  a.bias = bg; a.bias2 = bu; a.hidden = to;
  int rc = tiles_of(a, 2);
  if (!rc) rc = map_k(&maps.a[0], x, false, 128);
  if (!rc) rc = map_k(&maps.b[0], wg, false, a.ct / 2);
  if (!rc) rc = map_k(&maps.b[1], wu, false, a.ct / 2);
  if (!rc) rc = map_hidden(maps, to, m);
  if (!rc) rc = map_out(&maps.out[0], to.h, to.pitch, m);
  if (rc) return rc;
  return act == ACT_SILU ? launch<GATED, false, false, false, ACT_SILU>(maps, a, false, st) : launch<GATED, false, false, false, ACT_GELU>(maps, a, false, st);
}

int64_t fovi::tc_sum_rows(int64_t tokens) { return (tokens + 255) / 256 * 8; }

int fovi::tc_hidden_grad(const TcMatrix& dy, const TcMatrix& wd, const Hidden& from, int act, void* dg, void* du, float* sums, cudaStream_t st) {
  PtArgs a{};
  PtMaps maps{};
  const int64_t m = dy.rows;
  const int n = (int)wd.cols;
  a.tasks = 1; a.m[0] = (int)m; a.n[0] = n;
  a.kb0 = a.kb = (int)stages_of(dy.cols);
  a.splits = 1;
  a.ct = shape_of(&m, &n, 1, a.kb, 1, false).ct;
  a.hidden = from; a.sums = sums;
  int rc = tiles_of(a, 1);
  if (!rc) rc = map_k(&maps.a[0], dy, false, 128);
  if (!rc) rc = map_mn(&maps.b[0], wd);
  if (!rc) rc = map_hidden(maps, from, m);
  if (!rc) rc = map_out(&maps.out[0], dg, from.pitch, m);
  if (!rc) rc = map_out(&maps.out[1], du, from.pitch, m);
  if (rc) return rc;
  // The biases' sums of dg and du before these are rounded, which leaves one rounding of two in a bias's gradient, take 62 exchanges of lanes a chunk: 0.42 us a million hidden values
  // (16448 x 5120: 291 us, of the rounded ones 256), so up to 2^25 of them.
  if (sums && m * from.pitch <= 1 << 25)
    return act == ACT_SILU ? launch<GRAD, false, true, false, ACT_SILU, true>(maps, a, false, st) : launch<GRAD, false, true, false, ACT_GELU, true>(maps, a, false, st);
  return act == ACT_SILU ? launch<GRAD, false, true, false, ACT_SILU>(maps, a, false, st) : launch<GRAD, false, true, false, ACT_GELU>(maps, a, false, st);
}

// The cut of y = A B^T over `segments` pairs of matrices of k each, every one in whole stages: what a launch takes and what its workspace is counted by.
static TcShape linear_shape(int64_t m, int n, int64_t k, int segments) { return shape_of(&m, &n, 1, segments * stages_of(k), 1, true); }

int64_t fovi::tc_linear_bytes(int64_t m, int n, int64_t k, int segments) {
  const TcShape s = linear_shape(m, n, k, segments);
  return s.splits > 1 ? (int64_t)s.splits * m * ((n + 31) / 32 * 32) * 4 : 0;
}

int fovi::tc_linear(const TcMatrix& am, const TcMatrix& bm, const TcMatrix* a2, const TcMatrix* b2, bool b_mn, int m, int n, const void* bias, void* y, void* work, cudaStream_t st) {
  PtArgs a{};
  PtMaps maps{};
  a.tasks = 1; a.m[0] = m; a.n[0] = n; a.y[0] = y;
  a.kb0 = (int)stages_of(am.cols);
  a.kb = a.kb0 * (a2 ? 2 : 1);
  const TcShape s = linear_shape(m, n, am.cols, a2 ? 2 : 1);
  a.ct = s.ct; a.splits = s.splits; a.work = static_cast<float*>(work); a.bias = bias;
  int rc = tiles_of(a, 1);
  if (!rc) rc = map_k(&maps.a[0], am, false, 128);
  if (!rc) rc = b_mn ? map_mn(&maps.b[0], bm) : map_k(&maps.b[0], bm, false, a.ct / 2);
  if (!rc && a2) rc = map_k(&maps.a[1], *a2, false, 128);
  if (!rc && a2) rc = b_mn ? map_mn(&maps.b[1], *b2) : map_k(&maps.b[1], *b2, false, a.ct / 2);
  if (rc) return rc;
  rc = b_mn ? launch<STORE, false, true, false>(maps, a, false, st) : launch<STORE, false, false, false>(maps, a, false, st);
  return rc || a.splits == 1 ? rc : join(a, st);
}

// The cut follows from all the block's weights, so that a gradient has the same bits whichever are asked for.
static TcShape grads_shape(const TcTask* tasks, int n, int64_t rows) {
  int64_t m[GROUPS];
  int cols[GROUPS];
  for (int t = 0; t < n; ++t) { m[t] = tasks[t].m; cols[t] = tasks[t].n; }
  return shape_of(m, cols, n, stages_of(rows), 1, true);
}

int64_t fovi::tc_weight_grads_bytes(const TcTask* tasks, int n, int64_t rows) {
  const TcShape s = grads_shape(tasks, n, rows);
  if (s.splits == 1) return 0;
  int64_t bytes = 0;
  for (int t = 0; t < n; ++t) bytes += (int64_t)s.splits * tasks[t].m * ((tasks[t].n + 31) / 32 * 32) * 4;
  return bytes;
}

int fovi::tc_weight_grads(const TcTask* tasks, int n, int64_t rows, void* work, cudaStream_t st) {
  PtArgs a{};
  PtMaps maps{};
  const TcShape s = grads_shape(tasks, n, rows);
  a.ct = s.ct; a.splits = s.splits; a.work = static_cast<float*>(work);
  a.kb0 = a.kb = (int)stages_of(rows);
  int64_t at = 0;
  int rc = FOVI_OK;
  for (int t = 0; t < n && !rc; ++t) {
    if (!tasks[t].y) continue;
    const int i = a.tasks++;
    a.m[i] = tasks[t].m; a.n[i] = tasks[t].n; a.y[i] = tasks[t].y; a.part[i] = at;
    at += (int64_t)a.splits * tasks[t].m * ((tasks[t].n + 31) / 32 * 32);
    rc = map_mn(&maps.a[i], tasks[t].a);
    if (!rc) rc = map_mn(&maps.b[i], tasks[t].b);
  }
  if (rc || !a.tasks) return rc;
  rc = tiles_of(a, 1);
  if (!rc) rc = launch<STORE, true, true, false>(maps, a, false, st);
  return rc || a.splits == 1 ? rc : join(a, st);
}

int fovi::tc_int8(const TcMatrix& q, const TcMatrix& w, const float* scale, const float* wscale, const float* bias, void* y, int y_dtype, bool selftest, cudaStream_t st) {
  PtArgs a{};
  PtMaps maps{};
  const int64_t m = q.rows;
  const int n = (int)w.rows;
  a.tasks = 1; a.m[0] = (int)m; a.n[0] = n; a.y[0] = y; a.y_f32 = y_dtype == FOVI_F32;
  a.kb0 = a.kb = (int)((q.cols + 127) / 128);
  a.splits = 1;
  a.ct = shape_of(&m, &n, 1, a.kb, 1, false).ct;
  a.scale = scale; a.wscale = wscale; a.bias_f = bias;
  int rc = tiles_of(a, 1);
  if (!rc) rc = map_k(&maps.a[0], q, true, 128);
  if (!rc) rc = map_k(&maps.b[0], w, true, a.ct / 2);
  return rc ? rc : launch<SCALED, false, false, true>(maps, a, selftest, st);
}

extern "C" int fovi_product_check(void* stream) {
  auto st = reinterpret_cast<cudaStream_t>(stream);
  int* words[2];
  FOVI_CUDA(status_word(&words[0]));
  int rc = fovi::split_status(&words[1]), sites[2] = {0, 0};
  if (rc) return rc;
  for (int i = 0; i < 2; ++i) FOVI_CUDA(cudaMemcpyAsync(&sites[i], words[i], sizeof(int), cudaMemcpyDeviceToHost, st));
  FOVI_CUDA(cudaStreamSynchronize(st));
  if (!sites[0] && !sites[1]) return FOVI_OK;
  for (int i = 0; i < 2; ++i) FOVI_CUDA(cudaMemsetAsync(words[i], 0, sizeof(int), st));
  FOVI_CUDA(cudaStreamSynchronize(st));
  fovi::g_last_cuda_error = "token product: wait site " + std::to_string(sites[0] ? sites[0] : sites[1]) + " gave up";
  return FOVI_ERR_DEVICE_TIMEOUT;
}
