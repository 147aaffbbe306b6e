// Float32 matrix products on the tensor cores.
//
// A float32 value is the sum of three bf16 values exactly: the value rounded to 8 bits, what is left rounded to 8 bits, and the rest.  (Below 2^-110 the rest is below bf16's smallest value:
// such values are taken to 2^-134.)
// Of the nine products of two values' parts the six largest are taken; what is left out is at most 2^-24 of the product, a float32 product's own rounding.  The six are exact in the
// tensor cores, whose sums lose up to a unit of float32 at each step: so a sum runs over 64 of k only (24 steps), and the sums of 64 are added in registers with float32's rounding.
//   bound: six bf16 products for one, 375 of 2250 TFLOP/s, where the multiply-add units give 74.  1028 tokens, 384 x 1021 channels (one round of 40 tiles and less): projections 23 us,
//   hidden gradients 25, down 16, input gradients 15, weight gradients 24; on the multiply-add units 98 in all at their peak, and a training pass of 288 as measured (now 125).
// The kernel is that of product_tc.cu with these differences: a stage is 64 of k of all three parts of both operands (96 KB of a CTA, two stages), six products are taken from it, least
// first, and both accumulators in tensor memory take turns by stage; the epilogue warps add each to their registers (32 columns x up to four chunks a thread) under the next one's products.
#include <algorithm>

#include "product_pair.cuh"
#include "product_split.cuh"

using fovi::SplitMatrix;
using fovi::SplitProduct;
using fovi::SplitTask;

namespace {

__device__ int g_status;           // wait site at which a kernel gave up, see fovi_product_check: one word per device

enum { GATED = 0, GRAD = 1, STORE = 2 };
constexpr int EPI_WARPS = 8, PS_THREADS = (EPI_WARPS + 2) * 32, STAGES = 2, GROUPS = 3;
constexpr uint32_t PART = 16384, STAGE_BYTES = 6 * PART;            // three parts of 128 rows of A, and of up to 128 rows of B
constexpr uint32_t SCRATCH = 32 * 33 * 4;                           // of an epilogue warp: 32 rows x 32 columns (odd pitch), or 64 biases
constexpr uint32_t PS_SMEM = 1024 + 1024 + EPI_WARPS * SCRATCH + STAGES * STAGE_BYTES;
static_assert(PS_SMEM <= 227 * 1024 && SCRATCH * EPI_WARPS % 1024 == 0, "");

struct PsMaps { CUtensorMap a[GROUPS], b[GROUPS]; };                // of each task, or of each segment of k: [part][row][value]

struct PsArgs {
  int tasks, first[GROUPS + 1];            // tiles first[t] .. first[t + 1] - 1 belong to task t
  int n_mt[GROUPS], n_nt[GROUPS], m[GROUPS], n[GROUPS];
  float* y[GROUPS];
  int64_t part[GROUPS];                    // parts of k: where a task's begin in `work`
  int kb0, kb, splits, ct;                 // stages of the first segment of k, of all, parts; columns of a tile
  const float *bias, *bias2;
  float *g, *u; int64_t pitch;             // hidden values: their pitch, and the distance of two parts
  uint16_t *h, *dg, *du; int64_t part_of;
  float* work;
  int* status; uint32_t wait_limit;
};

struct PsHeader {
  uint64_t full[STAGES], empty[STAGES], acc_full[2], acc_empty[2], drain;
  uint32_t tmem_base;
  int abort_flag;
};

__device__ __forceinline__ void ps_load(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
               ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2) : "memory");
}

struct Tile { int task, mt, nt, k0, k1, split; };
__device__ __forceinline__ Tile tile_of(const PsArgs& a, int item) {
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

// The three parts of two values, as pairs.  The first two are rounded without leaving the range, so that a value that would round up to infinity keeps its rest, and infinity is the
// third part, which meets no other than a first one.
struct Parts { uint32_t w[3]; };
__device__ __forceinline__ uint32_t bf16_pair_finite(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
__device__ __forceinline__ float2 wide(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
__device__ __forceinline__ Parts cut_pair(float x, float y) {
  Parts p;
  float2 v = make_float2(x, y);
  p.w[0] = bf16_pair_finite(x, y);
  v = fma2(wide(p.w[0]), both(-1.f), v);
  p.w[1] = bf16_pair_finite(v.x, v.y);
  v = fma2(wide(p.w[1]), both(-1.f), v);
  p.w[2] = bf16_pair(v.x, v.y);
  return p;
}

// act(g) and act'(g)
template <int ACT> __device__ __forceinline__ float2 act32(float g) {
  if (ACT == fovi::ACT_SILU) {
    const float p = 1.f / (1.f + expf(-g)), a = g * p;
    return make_float2(a, fmaf(a, 1.f - p, p));
  }
  const float p = 0.5f * (1.f + erff(g * 0.70710678118654752f));
  return make_float2(g * p, fmaf(g * 0.39894228040143268f, expf(-0.5f * g * g), p));
}

template <int EPI, bool A_MN, bool B_MN, int ACT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PS_THREADS, 1) product_split_kernel(const __grid_constant__ PsMaps maps, const __grid_constant__ PsArgs a) {
  extern __shared__ unsigned char smem_raw[];
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  PsHeader* hdr = reinterpret_cast<PsHeader*>(smem_raw + (base - raw));
  const uint32_t stages0 = base + 1024u + EPI_WARPS * SCRATCH;
  volatile int* abort_flag = &hdr->abort_flag;
  const int warp = warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int rank = (int)pt_rank(), worker = blockIdx.x >> 1, workers = gridDim.x >> 1;
  const int half = a.ct / 2, total = a.first[a.tasks];

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(smem_u32(&hdr->full[s]), 1); mbar_init(smem_u32(&hdr->empty[s]), 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(smem_u32(&hdr->acc_full[i]), 1); mbar_init(smem_u32(&hdr->acc_empty[i]), 2 * EPI_WARPS); }
    mbar_init(smem_u32(&hdr->drain), 1);
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
    bool ok = true;
    for (int item = worker; item < total && ok; item += workers) {
      const Tile t = tile_of(a, item);
      const int m0 = t.mt * 256 + rank * 128, n0 = EPI == GATED ? t.nt * half : t.nt * a.ct + rank * half;
      for (int kb = t.k0; kb < t.k1; ++kb) {
        ok = mbar_wait_warp(smem_u32(&hdr->empty[s]), ph ^ 1u, abort_flag, a.status, 51, a.wait_limit);
        if (!ok) break;
        const int seg = kb >= a.kb0 ? 1 : 0, k = (kb - (seg ? a.kb0 : 0)) * 64;
        const CUtensorMap *ma = &maps.a[t.task + seg], *mb = &maps.b[EPI == GATED ? rank : t.task + seg];
        const uint32_t full = pt_map(smem_u32(&hdr->full[s]), 0), sa = stages0 + s * STAGE_BYTES, sb = sa + 3 * PART;
        if (elect_one()) {
          if (rank == 0) mbar_expect_tx(smem_u32(&hdr->full[s]), 6u * (PART + b_bytes));      // of both CTAs
#pragma unroll
          for (int p = 0; p < 3; ++p) {
            if (A_MN) {
              ps_load(sa + p * PART, ma, full, m0, k, p);
              ps_load(sa + p * PART + 8192u, ma, full, m0 + 64, k, p);
            } else {
              ps_load(sa + p * PART, ma, full, k, m0, p);
            }
            if (B_MN) {
              for (int j = 0; j < half; j += 64) ps_load(sb + p * PART + j * 128u, mb, full, n0 + j, k, p);
            } else {
              ps_load(sb + p * PART, mb, full, k, n0, p);
            }
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
      const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (A_MN ? 1u << 15 : 0u) | (B_MN ? 1u << 16 : 0u) | ((uint32_t)(a.ct >> 3) << 17) | (16u << 24);
      const uint64_t desc_a = smem_desc(0, A_MN ? 8192u : 16u, 1024u, 2u), desc_b = smem_desc(0, B_MN ? 8192u : 16u, 1024u, 2u);
      const uint32_t u_stages0 = warp_uniform(stages0), u_tmem = warp_uniform(tmem);
      uint32_t s = 0, ph = 0, acc = 0, aph = 0;
      bool ok = true;
      for (int item = worker; item < total && ok; item += workers) {
        const Tile t = tile_of(a, item);
        const int steps = warp_uniform(t.k1 - t.k0);
        for (int st = 0; st < steps; ++st) {
          ok = mbar_wait_warp(smem_u32(&hdr->acc_empty[acc]), aph ^ 1u, abort_flag, a.status, 52, a.wait_limit);
          if (ok) ok = mbar_wait_warp(smem_u32(&hdr->full[s]), ph, abort_flag, a.status, 53, a.wait_limit);
          if (!ok) break;
          tc_fence_after();
          const uint32_t sa = u_stages0 + s * STAGE_BYTES, d = u_tmem + acc * 256u;
          const uint64_t da = desc_a + (sa >> 4), db = desc_b + ((sa + 3 * PART) >> 4);
          if (elect_one()) {
            constexpr int PA[6] = {2, 0, 1, 1, 0, 0}, PB[6] = {0, 2, 1, 0, 1, 0};
#pragma unroll
            for (int q = 0; q < 6; ++q)
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                pt_mma<false>(d, da + PA[q] * (PART >> 4) + kk * (A_MN ? 128u : 2u), db + PB[q] * (PART >> 4) + kk * (B_MN ? 128u : 2u), idesc, (q | kk) ? 1u : 0u);
            pt_commit(smem_u32(&hdr->empty[s]));
            pt_commit(smem_u32(&hdr->acc_full[acc]));
          }
          __syncwarp();
          if (++s == STAGES) { s = 0; ph ^= 1u; }
          if (++acc == 2) { acc = 0; aph ^= 1u; }
        }
      }
      if (*abort_flag && elect_one()) {
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(&hdr->drain)) : "memory");
        for (uint32_t i = 0; i < (1u << 20); ++i)
          if (mbar_try_wait(smem_u32(&hdr->drain), 0)) break;
      }
    }
  } else {
    // ------------------------------------------------------------ sums of stages, epilogue
    const int quarter = warp & 3, turn = warp >> 2;
    float* scratch = reinterpret_cast<float*>(smem_raw + (base - raw) + 1024u + warp * SCRATCH);
    const int width = EPI == GATED ? half : a.ct;                     // columns of a tile; this warp's chunks of 32 are turn, turn + 2, ...
    constexpr int MINE = EPI == GATED ? 2 : 4, SETS = EPI == GATED ? 2 : 1;
    uint32_t acc = 0, aph = 0;
    bool lost = false;
    for (int item = worker; item < total && !lost; item += workers) {
      const Tile t = tile_of(a, item);
      const int row0 = t.mt * 256 + rank * 128 + quarter * 32, row = row0 + lane;
      const int M = a.m[t.task], N = a.n[t.task];
      const bool here = row < M;
      const int col0 = t.nt * width, end = EPI == STORE ? N : (int)a.pitch, chunks = min(width / 32, (end - col0 + 31) / 32);
      float2 sum[MINE][SETS][16];
#pragma unroll
      for (int c = 0; c < MINE; ++c)
#pragma unroll
        for (int q = 0; q < SETS; ++q)
#pragma unroll
          for (int i = 0; i < 16; ++i) sum[c][q][i] = both(0.f);
      for (int kb = t.k0; kb < t.k1; ++kb) {
        if (!mbar_wait_warp(smem_u32(&hdr->acc_full[acc]), aph, abort_flag, a.status, 54, a.wait_limit)) { lost = true; break; }
        tc_fence_after();
        const uint32_t t_base = tmem + ((uint32_t)(quarter * 32) << 16) + acc * 256u;
#pragma unroll
        for (int ci = 0; ci < MINE; ++ci) {
          const int c = turn + 2 * ci;
          if (c < chunks) {
#pragma unroll
            for (int q = 0; q < SETS; ++q) {
              uint32_t r[32];
              tc_ld32(t_base + q * half + 32 * c, r);
              tc_ld_wait();
              pt_loaded(r);
#pragma unroll
              for (int i = 0; i < 16; ++i) sum[ci][q][i] = add2(sum[ci][q][i], make_float2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])));
            }
          }
        }
        tc_fence_before();                         // (relaxed: see product_tc.cu)
        __syncwarp();
        if (lane == 0) asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(pt_map(smem_u32(&hdr->acc_empty[acc]), 0)) : "memory");
        if (++acc == 2) { acc = 0; aph ^= 1u; }
      }
      if (lost) break;
#pragma unroll
      for (int ci = 0; ci < MINE; ++ci) {
        const int c = turn + 2 * ci, c0 = col0 + 32 * c;
        if (c >= chunks) break;
        const int64_t at = (int64_t)row * a.pitch + c0;
        auto put_parts = [&](uint16_t* to, int i, const float* v) {       // of 16 columns from i on
          uint32_t w[3][8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const Parts p = cut_pair(v[2 * j], v[2 * j + 1]);
#pragma unroll
            for (int q = 0; q < 3; ++q) w[q][j] = p.w[q];
          }
#pragma unroll
          for (int q = 0; q < 3; ++q) st_global_32(to + q * a.part_of + at + i, w[q]);
        };
        auto put32 = [&](float* to, const float* v, int n) {
#pragma unroll
          for (int i = 0; i < n; i += 8) {
            uint32_t w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = __float_as_uint(v[i + j]);
            st_global_32(to + i, w);
          }
        };
        // 16 columns at a time, which registers hold beside the sums.
        if (EPI == GATED) {
          const int n = c0 + lane;
          __syncwarp();
          scratch[lane] = a.bias && n < N ? __ldg(a.bias + n) : 0.f;
          scratch[32 + lane] = a.bias2 && n < N ? __ldg(a.bias2 + n) : 0.f;
          __syncwarp();
#pragma unroll
          for (int i0 = 0; i0 < 32; i0 += 16) {
            float g[16], u[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int e = i0 + i;
              g[i] = (e & 1 ? sum[ci][0][e / 2].y : sum[ci][0][e / 2].x) + scratch[e];
              u[i] = (e & 1 ? sum[ci][SETS - 1][e / 2].y : sum[ci][SETS - 1][e / 2].x) + scratch[32 + e];
            }
            if (here) {
              if (a.g) { put32(a.g + at + i0, g, 16); put32(a.u + at + i0, u, 16); }
#pragma unroll
              for (int i = 0; i < 16; ++i) u[i] *= act32<ACT>(g[i]).x;
              put_parts(a.h, i0, u);
            }
          }
        } else if (EPI == GRAD) {
          if (here) {
#pragma unroll
            for (int i0 = 0; i0 < 32; i0 += 16) {
              float x[16], y[16];                  // g and u, then dg and du
#pragma unroll
              for (int i = 0; i < 16; i += 4) {
                *reinterpret_cast<float4*>(x + i) = *reinterpret_cast<const float4*>(a.g + at + i0 + i);
                *reinterpret_cast<float4*>(y + i) = *reinterpret_cast<const float4*>(a.u + at + i0 + i);
              }
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const int e = i0 + i;
                const float2 s = act32<ACT>(x[i]);
                const float dh = e & 1 ? sum[ci][0][e / 2].y : sum[ci][0][e / 2].x;
                x[i] = dh * y[i] * s.y;
                y[i] = dh * s.x;
              }
              put_parts(a.dg, i0, x);
              put_parts(a.du, i0, y);
            }
          }
        } else {
          float v[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = i & 1 ? sum[ci][0][i / 2].y : sum[ci][0][i / 2].x;
          if (a.splits > 1) {
            if (here) put32(a.work + a.part[t.task] + ((int64_t)t.split * M + row) * ((N + 31) / 32 * 32) + c0, v, 32);
            continue;
          }
          const float b = a.bias && c0 + lane < N ? __ldg(a.bias + c0 + lane) : 0.f;
          float* y = a.y[t.task];
          if (N % 8 == 0) {
            __syncwarp();
            scratch[lane] = b;
            __syncwarp();
            if (here) {
#pragma unroll
              for (int i = 0; i < 32; i += 8) {
                uint32_t w[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] = __float_as_uint(v[i + j] + scratch[i + j]);
                if (c0 + i < N) st_global_32(y + (int64_t)row * N + c0 + i, w);
              }
            }
          } else {                               // through the warp's scratch, so that lanes write neighbouring columns
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 32; ++i) scratch[lane * 33 + i] = v[i];
            __syncwarp();
            if (c0 + lane < N) {
              const int rows = min(32, M - row0);
#pragma unroll 8
              for (int r = 0; r < rows; ++r) y[(int64_t)(row0 + r) * N + c0 + lane] = scratch[r * 33 + lane] + b;
            }
          }
          __syncwarp();
        }
      }
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
struct JoinArgs { const float* part[GROUPS]; float* y[GROUPS]; int64_t m[GROUPS]; int n[GROUPS], splits; const float* bias; };
__global__ void __launch_bounds__(256) product_split_join_kernel(const __grid_constant__ JoinArgs a) {
  const int t = blockIdx.y, n = a.n[t];
  const uint32_t pitch = (n + 31) / 32 * 32, per = pitch / 4;
  const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x, row = i >> 32 ? i / per : (uint32_t)i / per;
  const int c = (int)(i - row * per) * 4;
  const int64_t m = a.m[t];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if ((int64_t)row >= m || c >= n) return;
  const float* from = a.part[t] + row * pitch + c;
  float s[4] = {};
#pragma unroll 4
  for (int p = 0; p < a.splits; ++p) {
    float4 v;
    asm volatile("ld.global.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(from + p * m * pitch) : "memory");
    s[0] += v.x; s[1] += v.y; s[2] += v.z; s[3] += v.w;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (a.bias && c + e < n) s[e] += __ldg(a.bias + c + e);
  float* to = a.y[t] + (int64_t)row * n + c;
  if (n % 4 == 0) {
    *reinterpret_cast<float4*>(to) = make_float4(s[0], s[1], s[2], s[3]);
  } else {
    for (int e = 0; e < 4 && c + e < n; ++e) to[e] = s[e];
  }
}

struct CutArgs { SplitTask t[fovi::SPLITS_MOST]; };
// A thread for eight neighbouring values of a row.
__global__ void __launch_bounds__(256) cut_kernel(const __grid_constant__ CutArgs a) {
  const SplitTask& t = a.t[blockIdx.y];
  const uint32_t per = (uint32_t)(t.to.pitch / 8);
  const uint64_t all = t.to.rows * per;
  const int64_t part = t.to.rows * t.to.pitch;
  const bool vec = t.stride % 4 == 0 && (reinterpret_cast<uintptr_t>(t.x) & 15) == 0;
  uint16_t* to = static_cast<uint16_t*>(t.to.p);
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (uint64_t)gridDim.x * 256) {
    const uint64_t r = i >> 32 ? i / per : (uint32_t)i / per;
    const int64_t c = 8 * (int64_t)(i - r * per);
    const float* x = t.x + r * t.stride + c;
    float v[8];
    if (vec && c + 8 <= t.to.cols) {
      const float4 lo = __ldg(reinterpret_cast<const float4*>(x)), hi = __ldg(reinterpret_cast<const float4*>(x) + 1);
      v[0] = lo.x; v[1] = lo.y; v[2] = lo.z; v[3] = lo.w; v[4] = hi.x; v[5] = hi.y; v[6] = hi.z; v[7] = hi.w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = c + j < t.to.cols ? __ldg(x + j) : 0.f;
    }
    uint32_t w[3][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const Parts p = cut_pair(v[2 * j], v[2 * j + 1]);
#pragma unroll
      for (int q = 0; q < 3; ++q) w[q][j] = p.w[q];
    }
#pragma unroll
    for (int q = 0; q < 3; ++q) *reinterpret_cast<uint4*>(to + q * part + r * t.to.pitch + c) = make_uint4(w[q][0], w[q][1], w[q][2], w[q][3]);
  }
}

// ------------------------------------------------------------------------------------------------------------ host
int pairs() { return std::max(1, fovi::sm_count() / 2); }
int64_t stages_of(int64_t k) { return (k + 63) / 64; }

struct Shape { int ct, splits; };
// The cut with the least time by a count of clocks, as in product_tc.cu: 12 clocks a column and stage, about 3000 for a tile's start and end, and for k in parts their way through memory.
Shape shape_of(const int64_t* m, const int* n, int tasks, int64_t kb, int share, bool may_split) {
  Shape best{256, 1};
  double least = 1e300;
  const int64_t at_once = pairs();
  for (int ct = 256; ct >= 64; ct -= 64) {
    int64_t tiles = 0, values = 0;
    for (int t = 0; t < tasks; ++t) {
      tiles += (m[t] + 255) / 256 * ((n[t] * (int64_t)share + ct - 1) / ct);
      values += m[t] * ((n[t] + 31) / 32 * 32);
    }
    for (int s = 1; s <= (may_split ? 32 : 1) && (s == 1 || kb / s >= 2); ++s) {
      const double ways = s > 1 ? 5000 + (double)values * s * 8 / 3400 : 0;
      if (ways >= least) break;
      const double clocks = ways + (double)((tiles * s + at_once - 1) / at_once) * ((double)((kb + s - 1) / s) * std::max(12 * ct, 1500) + 3000);
      if (clocks < least) { least = clocks; best = {ct, s}; }
    }
  }
  return best;
}

int map_k(CUtensorMap* m, const SplitMatrix& x, int rows) {
  return fovi::encode_3d(m, x.p, (uint64_t)x.cols, (uint64_t)x.rows, 3, (uint64_t)x.pitch * 2, (uint64_t)(x.rows * x.pitch) * 2, 64, (uint32_t)rows, 1, true);
}
int map_mn(CUtensorMap* m, const SplitMatrix& x) {
  return fovi::encode_3d(m, x.p, (uint64_t)x.cols, (uint64_t)x.rows, 3, (uint64_t)x.pitch * 2, (uint64_t)(x.rows * x.pitch) * 2, 64, 64, 1, true);
}

template <int EPI, bool A_MN, bool B_MN, int ACT = 0> int launch(const PsMaps& maps, PsArgs& a, cudaStream_t st) {
  int rc = fovi::split_status(&a.status);
  if (rc) return rc;
  a.wait_limit = WAIT_LIMIT;
  const int grid = 2 * std::min(a.first[a.tasks], pairs());
  auto kernel = product_split_kernel<EPI, A_MN, B_MN, ACT>;
  static std::atomic<uint64_t> done{0};
  FOVI_CUDA(allow_shared(kernel, (int)PS_SMEM, done));
  FOVI_CUDA(fovi::launch_pdl(kernel, grid, PS_THREADS, PS_SMEM, st, maps, a));
  return fovi::after_launch("product_split_kernel");
}

int tiles_of(PsArgs& a, int share) {
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

int join(const PsArgs& a, cudaStream_t st) {
  JoinArgs j{};
  int64_t threads = 0;
  j.splits = a.splits;
  j.bias = a.bias;
  for (int t = 0; t < a.tasks; ++t) {
    j.part[t] = a.work + a.part[t]; j.y[t] = a.y[t]; j.m[t] = a.m[t]; j.n[t] = a.n[t];
    threads = std::max(threads, (int64_t)a.m[t] * ((a.n[t] + 31) / 32 * 8));
  }
  FOVI_CUDA(fovi::launch_pdl(product_split_join_kernel, dim3((unsigned)((threads + 255) / 256), a.tasks), 256, 0, st, j));
  return fovi::after_launch("product_split_join_kernel");
}

int64_t part_bytes(const int64_t* m, const int* n, int tasks, int splits) {
  int64_t bytes = 0;
  for (int t = 0; splits > 1 && t < tasks; ++t) bytes += (int64_t)splits * m[t] * ((n[t] + 31) / 32 * 32) * 4;
  return bytes;
}

// The cut follows from all the block's weights, so that a gradient has the same bits whichever are asked for.
Shape grads_shape(const SplitProduct* tasks, int n, int64_t rows, int64_t* bytes) {
  int64_t m[GROUPS];
  int cols[GROUPS];
  for (int t = 0; t < n; ++t) { m[t] = tasks[t].m; cols[t] = tasks[t].n; }
  const Shape s = shape_of(m, cols, n, stages_of(rows), 1, true);
  *bytes = part_bytes(m, cols, n, s.splits);
  return s;
}

}  // namespace

int fovi::split_status(int** word) {
  static std::atomic<int*> known[64];
  FOVI_CUDA(word_of(word, g_status, known));
  return FOVI_OK;
}

int fovi::split_matrices(const SplitTask* t, int n, cudaStream_t st) {
  CutArgs a{};
  int64_t most = 0;
  for (int i = 0; i < n; ++i) {
    a.t[i] = t[i];
    most = std::max(most, t[i].to.rows * (t[i].to.pitch / 8));
  }
  cut_kernel<<<dim3((unsigned)std::min<int64_t>((most + 255) / 256, 8 * fovi::sm_count()), n), 256, 0, st>>>(a);
  return fovi::after_launch("cut_kernel");
}

int fovi::split_gated(const SplitMatrix& x, const SplitMatrix& wg, const SplitMatrix& wu, const float* bg, const float* bu, int act, float* g, float* u, const SplitMatrix& h,
                      cudaStream_t st) {
  PsArgs a{};
  PsMaps maps{};
  const int64_t m = x.rows;
  const int n = (int)wg.rows;
  a.tasks = 1; a.m[0] = (int)m; a.n[0] = n;
  a.kb0 = a.kb = (int)stages_of(x.cols);
  a.splits = 1;
  a.ct = shape_of(&m, &n, 1, a.kb, 2, false).ct;
  a.bias = bg; a.bias2 = bu; a.g = g; a.u = u; a.pitch = h.pitch; a.h = static_cast<uint16_t*>(h.p); a.part_of = h.rows * h.pitch;
  int rc = tiles_of(a, 2);
  if (!rc) rc = map_k(&maps.a[0], x, 128);
  if (!rc) rc = map_k(&maps.b[0], wg, a.ct / 2);
  if (!rc) rc = map_k(&maps.b[1], wu, a.ct / 2);
  if (rc) return rc;
  return act == ACT_SILU ? launch<GATED, false, false, ACT_SILU>(maps, a, st) : launch<GATED, false, false, ACT_GELU>(maps, a, st);
}

int fovi::split_hidden_grad(const SplitMatrix& dy, const SplitMatrix& wd, const float* g, const float* u, int act, const SplitMatrix& dg, const SplitMatrix& du, cudaStream_t st) {
  PsArgs a{};
  PsMaps maps{};
  const int64_t m = dy.rows;
  const int n = (int)wd.cols;
  a.tasks = 1; a.m[0] = (int)m; a.n[0] = n;
  a.kb0 = a.kb = (int)stages_of(dy.cols);
  a.splits = 1;
  a.ct = shape_of(&m, &n, 1, a.kb, 1, false).ct;
  a.g = const_cast<float*>(g); a.u = const_cast<float*>(u); a.pitch = dg.pitch; a.part_of = dg.rows * dg.pitch;
  a.dg = static_cast<uint16_t*>(dg.p); a.du = static_cast<uint16_t*>(du.p);
  int rc = tiles_of(a, 1);
  if (!rc) rc = map_k(&maps.a[0], dy, 128);
  if (!rc) rc = map_mn(&maps.b[0], wd);
  if (rc) return rc;
  return act == ACT_SILU ? launch<GRAD, false, true, ACT_SILU>(maps, a, st) : launch<GRAD, false, true, ACT_GELU>(maps, a, st);
}

// As in product_tc.cu: one cut for a launch and for its workspace.
static Shape linear_shape(int64_t m, int n, int64_t k, int segments) { return shape_of(&m, &n, 1, segments * stages_of(k), 1, true); }

int64_t fovi::split_linear_bytes(int64_t m, int n, int64_t k, int segments) { return part_bytes(&m, &n, 1, linear_shape(m, n, k, segments).splits); }

int fovi::split_linear(const SplitMatrix& am, const SplitMatrix& bm, const SplitMatrix* a2, const SplitMatrix* b2, bool b_mn, int m, int n, const float* bias, float* y, void* work,
                       cudaStream_t st) {
  PsArgs a{};
  PsMaps maps{};
  a.tasks = 1; a.m[0] = m; a.n[0] = n; a.y[0] = y;
  a.kb0 = (int)stages_of(am.cols);
  a.kb = a.kb0 * (a2 ? 2 : 1);
  const Shape s = linear_shape(m, n, am.cols, a2 ? 2 : 1);
  a.ct = s.ct; a.splits = s.splits; a.work = static_cast<float*>(work); a.bias = bias;
  int rc = tiles_of(a, 1);
  if (!rc) rc = map_k(&maps.a[0], am, 128);
  if (!rc) rc = b_mn ? map_mn(&maps.b[0], bm) : map_k(&maps.b[0], bm, a.ct / 2);
  if (!rc && a2) rc = map_k(&maps.a[1], *a2, 128);
  if (!rc && a2) rc = b_mn ? map_mn(&maps.b[1], *b2) : map_k(&maps.b[1], *b2, a.ct / 2);
  if (rc) return rc;
  rc = b_mn ? launch<STORE, false, true>(maps, a, st) : launch<STORE, false, false>(maps, a, st);
  return rc || a.splits == 1 ? rc : join(a, st);
}

int64_t fovi::split_weight_grads_bytes(const SplitProduct* tasks, int n, int64_t rows) {
  int64_t bytes;
  grads_shape(tasks, n, rows, &bytes);
  return bytes;
}

int fovi::split_weight_grads(const SplitProduct* tasks, int n, int64_t rows, void* work, cudaStream_t st) {
  PsArgs a{};
  PsMaps maps{};
  int64_t bytes, at = 0;
  const Shape s = grads_shape(tasks, n, rows, &bytes);
  a.ct = s.ct; a.splits = s.splits; a.work = static_cast<float*>(work);
  a.kb0 = a.kb = (int)stages_of(rows);
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
  if (!rc) rc = launch<STORE, true, true>(maps, a, st);
  return rc || a.splits == 1 ? rc : join(a, st);
}
