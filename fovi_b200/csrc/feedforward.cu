// Gated feed-forward block on tokens x [tokens, C]:
//   g = x Wg^T + bg,  u = x Wu^T + bu,  h = act(g) u,  y = h Wd^T + bd          Wg, Wu [F, C], Wd [O, F]; act(g) = g s(g) (s: logistic) or g Phi(g) (Phi: normal distribution)
// and, from g and u in 24 bits and h in bf16 (float32: in 32, h in parts), which the forward pass keeps, its gradients
//   dh = dy Wd,  dg = dh u act'(g),  du = dh act(g),  dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x,  dWd = dy^T h,  and column sums of dg, du, dy for the biases.
// bf16: sums are float32; h, dg and du are rounded to bf16 between the products, as the tensor cores take them (few tokens without gradients: h as two bf16 values).  With 24 bits of g and u
// what gradients lose by them is below those roundings; 16 would put two more into each.
#include <algorithm>

#include "product_few.cuh"
#include "product_split.cuh"
#include "product_tc.cuh"

using fovi::Hidden;
using fovi::SplitMatrix;
using fovi::SplitProduct;
using fovi::SplitTask;
using fovi::TcMatrix;
using fovi::TcTask;

namespace {

// Column sums of up to three matrices in a fixed order: parts of strips of rows, then the parts of each column; two launches for all.
struct SumTask { const void* x; int64_t rows, pitch; int n; float* part; int parts; int64_t part_pitch; void* out; bool bf16; };      // part: given (x null), or to be made; bf16: x's type
struct SumTasks { SumTask t[3]; };
constexpr int SUM_COLS = 256, STRIPS = 512;

// A block takes 256 columns of a strip of rows, a lane 8 neighbouring ones, its 8 warps a row each at a time.
template <typename T> __device__ __forceinline__ void column_parts(const SumTask& t, float (&red)[8][SUM_COLS + 8]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = blockIdx.x * SUM_COLS + 8 * lane;
  const int64_t r0 = t.rows * blockIdx.y / t.parts, r1 = t.rows * (blockIdx.y + 1) / t.parts;
  const T* x = static_cast<const T*>(t.x) + c;
  float s[8] = {};
  const bool whole = c + 8 <= t.n && t.pitch % (16 / sizeof(T)) == 0 && (reinterpret_cast<uintptr_t>(t.x) & 15) == 0;
  if (whole) {
#pragma unroll 4
    for (int64_t r = r0 + warp; r < r1; r += 8) {
      uint4 w[sizeof(T) / 2];
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = __ldg(reinterpret_cast<const uint4*>(x + r * t.pitch) + i);
      const T* v = reinterpret_cast<const T*>(w);
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] += (float)v[i];
    }
  } else {
    for (int64_t r = r0 + warp; r < r1; r += 8)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + i < t.n) s[i] += ld_as_float(x + r * t.pitch + i);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) red[warp][8 * lane + i] = s[i];
  __syncthreads();
  const int col = blockIdx.x * SUM_COLS + threadIdx.x;
  if (col >= t.n) return;
  float sum = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) sum += red[w][threadIdx.x];
  t.part[blockIdx.y * t.part_pitch + col] = sum;
}
__global__ void __launch_bounds__(256) column_parts_kernel(const __grid_constant__ SumTasks tasks) {
  __shared__ float red[8][SUM_COLS + 8];
  const SumTask& t = tasks.t[blockIdx.z];
  if (!t.x || (int)blockIdx.y >= t.parts || blockIdx.x * SUM_COLS >= t.n) return;
  if (t.bf16) column_parts<__nv_bfloat16>(t, red);
  else column_parts<float>(t, red);
}
template <typename T>
__global__ void __launch_bounds__(1024) column_join_kernel(const __grid_constant__ SumTasks tasks) {
  const SumTask& t = tasks.t[blockIdx.y];
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  if (!t.out || blockIdx.x * 32 >= t.n) return;
  float s = 0.f;
  if (c < t.n)
    for (int p = w; p < t.parts; p += 32) s += t.part[p * t.part_pitch + c];
  red[w][lane] = s;
  __syncthreads();
  if (w || c >= t.n) return;
  s = 0.f;
  for (int i = 0; i < 32; ++i) s += red[i][lane];
  static_cast<T*>(t.out)[c] = from_float<T>(s);
}
SumTask sum_task(const void* x, int64_t rows, int n, int64_t pitch, float* part, void* out, bool bf16) {
  return {x, rows, pitch, n, part, (int)std::max<int64_t>(1, std::min<int64_t>(STRIPS, rows / 32)), n, out, bf16};
}
// T: the sums' type.
template <typename T> int column_sums(const SumTasks& tasks, cudaStream_t st) {
  int wide = 0, strips = 0, most = 0;
  for (const SumTask& t : tasks.t) {
    if (t.out) most = std::max(most, t.n);
    if (t.out && t.x) { wide = std::max(wide, t.n); strips = std::max(strips, t.parts); }
  }
  if (wide) {
    column_parts_kernel<<<dim3((wide + SUM_COLS - 1) / SUM_COLS, strips, 3), 256, 0, st>>>(tasks);
    const int rc = fovi::after_launch("column_parts_kernel");
    if (rc) return rc;
  }
  if (!most) return FOVI_OK;
  column_join_kernel<T><<<dim3((most + 31) / 32, 3), 1024, 0, st>>>(tasks);
  return fovi::after_launch("column_join_kernel");
}

int64_t pitch_of(int F) { return ((int64_t)F + 31) / 32 * 32; }
// Where the parts of a bf16 block's buffer for the hidden values lie.
Hidden hidden_at(void* p, int64_t M, int F, bool saved) {
  Hidden h{};
  h.pitch = pitch_of(F);
  h.h = p;
  if (saved) {
    h.high = static_cast<uint16_t*>(p) + M * h.pitch;
    h.low = reinterpret_cast<uint8_t*>(h.high + 2 * M * h.pitch);
  }
  return h;
}

struct Block {
  const void *x, *wg, *wu, *wd, *bg, *bu, *bd;
  int64_t M, xs, gs, us, ds; int C, F, O, act;
};

// The parts of a workspace, each on a boundary of 256 bytes.
int64_t padded(int64_t bytes) { return (bytes + 255) / 256 * 256; }

int forward_bf16(const Block& b, void* y, const Hidden& hid, void* work, cudaStream_t st) {
  if (!hid.high && fovi::few_block(b.M, b.C, b.F, b.O)) {
    const int rc = fovi::few_gated({b.x, b.xs}, {b.wg, b.gs}, {b.wu, b.us}, (int)b.M, b.F, b.C, b.bg, b.bu, b.act, {hid.h, hid.pitch}, st);
    return rc ? rc : fovi::few_down({hid.h, hid.pitch}, {b.wd, b.ds}, (int)b.M, b.O, b.F, b.bd, y, st);
  }
  const TcMatrix x{b.x, b.M, b.C, b.xs}, wg{b.wg, b.F, b.C, b.gs}, wu{b.wu, b.F, b.C, b.us}, wd{b.wd, b.O, b.F, b.ds}, h{hid.h, b.M, b.F, hid.pitch};
  const int rc = fovi::tc_gated(x, wg, wu, b.bg, b.bu, b.act, hid, st);
  return rc ? rc : fovi::tc_linear(h, wd, nullptr, nullptr, false, (int)b.M, b.O, b.bd, y, work, st);
}

struct Grads { const void* dy; int64_t dys; void *dx, *dwg, *dwu, *dwd, *dbg, *dbu, *dbd; };

// ------------------------------------------------------------------------------------------------------------ float32 on the tensor cores
// Where the float32 block's operands in parts lie: one behind the other from `at` on.
struct Cut {
  char* at;
  int64_t used = 0;
  SplitMatrix take(int64_t rows, int64_t cols, int64_t pitch) {
    const SplitMatrix m{at ? at + used : nullptr, rows, cols, pitch};
    used += padded(3 * rows * pitch * 2);
    return m;
  }
  SplitMatrix take(int64_t rows, int64_t cols) { return take(rows, cols, fovi::split_pitch(cols)); }
};
struct SplitForward { SplitMatrix x, wg, wu, wd, h; int64_t parts, bytes; };
SplitForward split_forward_at(const Block& b, bool saved, char* work) {
  Cut c{work};
  SplitForward f;
  f.x = c.take(b.M, b.C);
  f.wg = c.take(b.F, b.C);
  f.wu = c.take(b.F, b.C);
  f.wd = c.take(b.O, b.F);
  if (!saved) f.h = c.take(b.M, b.F, pitch_of(b.F));
  f.parts = c.used;
  f.bytes = c.used + fovi::split_linear_bytes(b.M, b.O, b.F, 1);
  return f;
}
// saved: g, u, then h in parts.
SplitMatrix saved_parts(void* saved, const Block& b) {
  const int64_t pitch = pitch_of(b.F);
  return {static_cast<char*>(saved) + 8 * b.M * pitch, b.M, b.F, pitch};
}

int forward_split(const Block& b, void* y, void* saved, char* work, cudaStream_t st) {
  if (!saved && fovi::few_float(b.M, b.C, b.F, b.O)) {
    auto f = [](const void* p) { return static_cast<const float*>(p); };
    return fovi::few_block32(f(b.x), b.xs, f(b.wg), b.gs, f(b.wu), b.us, f(b.wd), b.ds, (int)b.M, b.C, b.F, b.O, f(b.bg), f(b.bu), f(b.bd), b.act, reinterpret_cast<float*>(work),
                             pitch_of(b.F), static_cast<float*>(y), st);
  }
  SplitForward f = split_forward_at(b, saved != nullptr, work);
  float *g = static_cast<float*>(saved), *u = saved ? g + b.M * pitch_of(b.F) : nullptr;
  if (saved) f.h = saved_parts(saved, b);
  const SplitTask cut[4] = {{static_cast<const float*>(b.x), b.xs, f.x}, {static_cast<const float*>(b.wg), b.gs, f.wg}, {static_cast<const float*>(b.wu), b.us, f.wu},
                            {static_cast<const float*>(b.wd), b.ds, f.wd}};
  int rc = fovi::split_matrices(cut, 4, st);
  if (!rc) rc = fovi::split_gated(f.x, f.wg, f.wu, static_cast<const float*>(b.bg), static_cast<const float*>(b.bu), b.act, g, u, f.h, st);
  return rc ? rc : fovi::split_linear(f.h, f.wd, nullptr, nullptr, false, (int)b.M, b.O, static_cast<const float*>(b.bd), static_cast<float*>(y), work + f.parts, st);
}

struct SplitBackward { SplitMatrix x, wg, wu, wd, dy, dg, du; SplitProduct t[3]; int64_t parts, bytes; };
SplitBackward split_backward_at(const Block& b, const SplitMatrix& h, char* work) {
  Cut c{work};
  SplitBackward f;
  f.x = c.take(b.M, b.C);
  f.wg = c.take(b.F, b.C);
  f.wu = c.take(b.F, b.C);
  f.wd = c.take(b.O, b.F);
  f.dy = c.take(b.M, b.O);
  f.dg = c.take(b.M, b.F, pitch_of(b.F));
  f.du = c.take(b.M, b.F, pitch_of(b.F));
  f.t[0] = {f.dg, f.x, b.F, b.C, nullptr};
  f.t[1] = {f.du, f.x, b.F, b.C, nullptr};
  f.t[2] = {f.dy, h, b.O, b.F, nullptr};
  f.parts = c.used;
  f.bytes = c.used + std::max({fovi::split_linear_bytes(b.M, b.C, b.F, 2), fovi::split_weight_grads_bytes(f.t, 3, b.M), STRIPS * (2 * (int64_t)b.F + b.O) * 4});
  return f;
}

int backward_split(const Block& b, const void* saved, const Grads& g, char* work, cudaStream_t st) {
  SplitBackward f = split_backward_at(b, saved_parts(const_cast<void*>(saved), b), work);
  const float *gv = static_cast<const float*>(saved), *uv = gv + b.M * pitch_of(b.F);
  float* parts = reinterpret_cast<float*>(work + f.parts);
  const bool hidden = g.dx || g.dwg || g.dwu || g.dbg || g.dbu;
  SplitTask cut[5];
  int n = 0;
  if (hidden || g.dwd) cut[n++] = {static_cast<const float*>(g.dy), g.dys, f.dy};
  if (hidden) cut[n++] = {static_cast<const float*>(b.wd), b.ds, f.wd};
  if (g.dwg || g.dwu) cut[n++] = {static_cast<const float*>(b.x), b.xs, f.x};
  if (g.dx) {
    cut[n++] = {static_cast<const float*>(b.wg), b.gs, f.wg};
    cut[n++] = {static_cast<const float*>(b.wu), b.us, f.wu};
  }
  int rc = n ? fovi::split_matrices(cut, n, st) : FOVI_OK;
  if (!rc && hidden) rc = fovi::split_hidden_grad(f.dy, f.wd, gv, uv, b.act, f.dg, f.du, st);
  if (!rc && g.dx) rc = fovi::split_linear(f.dg, f.wg, &f.du, &f.wu, true, (int)b.M, b.C, nullptr, static_cast<float*>(g.dx), parts, st);
  f.t[0].y = static_cast<float*>(g.dwg); f.t[1].y = static_cast<float*>(g.dwu); f.t[2].y = static_cast<float*>(g.dwd);
  if (!rc) rc = fovi::split_weight_grads(f.t, 3, b.M, parts, st);
  if (rc) return rc;
  // The biases' sums: of dg and du over the rows of all three parts, of dy as it is.
  SumTasks tasks{};
  float* const at[3] = {parts, parts + (int64_t)STRIPS * b.F, parts + 2 * (int64_t)STRIPS * b.F};
  if (g.dbg) tasks.t[0] = sum_task(f.dg.p, 3 * b.M, b.F, f.dg.pitch, at[0], g.dbg, true);
  if (g.dbu) tasks.t[1] = sum_task(f.du.p, 3 * b.M, b.F, f.du.pitch, at[1], g.dbu, true);
  if (g.dbd) tasks.t[2] = sum_task(g.dy, b.M, b.O, g.dys, at[2], g.dbd, false);
  return column_sums<float>(tasks, st);
}

// The three weight gradients as products over the tokens.
void weight_tasks(const Block& b, const Hidden& hid, const Grads& g, const void* dg, const void* du, TcTask (&t)[3]) {
  t[0] = TcTask{{dg, b.M, b.F, hid.pitch}, {b.x, b.M, b.C, b.xs}, b.F, b.C, g.dwg};
  t[1] = TcTask{{du, b.M, b.F, hid.pitch}, {b.x, b.M, b.C, b.xs}, b.F, b.C, g.dwu};
  t[2] = TcTask{{g.dy, b.M, b.O, g.dys}, {hid.h, b.M, b.F, hid.pitch}, b.O, b.F, g.dwd};
}

// Work of a bf16 backward pass: dg, du; then, one after another in the same place, the parts of dx, of the weight gradients, and of the biases' sums of dy.  The sums of
// dg and du, which the first kernel leaves, have a place of their own.
struct BackWork { int64_t sums, parts, bytes; };
BackWork back_work(const Block& b, int64_t pitch) {
  TcTask t[3];
  weight_tasks(b, Hidden{}, Grads{}, nullptr, nullptr, t);
  BackWork w;
  w.sums = padded(2 * b.M * pitch * 2);
  w.parts = w.sums + padded(fovi::tc_sum_rows(b.M) * 2 * pitch * 4);
  w.bytes = w.parts + std::max({fovi::tc_linear_bytes(b.M, b.C, b.F, 2), fovi::tc_weight_grads_bytes(t, 3, b.M), (int64_t)STRIPS * b.O * 4});
  return w;
}

int backward_bf16(const Block& b, const Hidden& hid, const Grads& g, char* work, cudaStream_t st) {
  const BackWork at = back_work(b, hid.pitch);
  __nv_bfloat16 *dg = reinterpret_cast<__nv_bfloat16*>(work), *du = dg + b.M * hid.pitch;
  float *sums = reinterpret_cast<float*>(work + at.sums), *parts = reinterpret_cast<float*>(work + at.parts);
  const TcMatrix dy{g.dy, b.M, b.O, g.dys}, wg{b.wg, b.F, b.C, b.gs}, wu{b.wu, b.F, b.C, b.us}, wd{b.wd, b.O, b.F, b.ds};
  const TcMatrix dgm{dg, b.M, b.F, hid.pitch}, dum{du, b.M, b.F, hid.pitch};
  int rc;
  if (g.dx || g.dwg || g.dwu || g.dbg || g.dbu) {
    if ((rc = fovi::tc_hidden_grad(dy, wd, hid, b.act, dg, du, g.dbg || g.dbu ? sums : nullptr, st))) return rc;
  }
  if (g.dx && (rc = fovi::tc_linear(dgm, wg, &dum, &wu, true, (int)b.M, b.C, nullptr, g.dx, parts, st))) return rc;
  TcTask t[3];
  weight_tasks(b, hid, g, dg, du, t);
  if ((rc = fovi::tc_weight_grads(t, 3, b.M, parts, st))) return rc;
  SumTasks tasks{};
  const int rows = (int)fovi::tc_sum_rows(b.M);
  if (g.dbg) tasks.t[0] = SumTask{nullptr, 0, 0, b.F, sums, rows, 2 * hid.pitch, g.dbg, false};
  if (g.dbu) tasks.t[1] = SumTask{nullptr, 0, 0, b.F, sums + hid.pitch, rows, 2 * hid.pitch, g.dbu, false};
  if (g.dbd) tasks.t[2] = sum_task(g.dy, b.M, b.O, g.dys, parts, g.dbd, true);
  return column_sums<__nv_bfloat16>(tasks, st);
}

// Copies of bf16 matrices whose rows do not start on 16-byte boundaries, to where they do, up to five in one launch.  A thread for eight values of a row.
struct PadTask { const uint16_t* x; int64_t stride; uint16_t* to; int64_t rows, cols, pitch; };
struct PadArgs { PadTask t[5]; };
__global__ void __launch_bounds__(256) pad_kernel(const __grid_constant__ PadArgs a) {
  const PadTask& t = a.t[blockIdx.y];
  const uint32_t per = (uint32_t)(t.pitch / 8);
  const uint64_t all = t.rows * per;
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (uint64_t)gridDim.x * 256) {
    const int64_t r = i >> 32 ? i / per : (uint32_t)i / per, c = 8 * (int64_t)(i - r * per);
    const uint16_t* x = t.x + r * t.stride + c;
    uint32_t w[4] = {};
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j < t.cols) w[j / 2] |= (uint32_t)__ldg(x + j) << (16 * (j & 1));
    *reinterpret_cast<uint4*>(t.to + r * t.pitch + c) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
int64_t pad_bytes(int64_t rows, int64_t cols) { return padded(rows * fovi::split_pitch(cols) * 2); }
int64_t pads_bytes(int64_t M, int64_t C, int64_t F, int64_t O, bool backward) {
  return pad_bytes(M, C) + 2 * pad_bytes(F, C) + pad_bytes(O, F) + (backward ? pad_bytes(M, O) : 0);
}
bool boundaries(const Block& b, const Grads* g) {
  return fovi::tc_takes(b.x, b.xs, 2) && fovi::tc_takes(b.wg, b.gs, 2) && fovi::tc_takes(b.wu, b.us, 2) && fovi::tc_takes(b.wd, b.ds, 2) && (!g || fovi::tc_takes(g->dy, g->dys, 2));
}
// The block (and dy) with copies in `at` for what does not lie on boundaries; moves `at` behind them.
int pad(Block& b, Grads* g, char*& at, cudaStream_t st) {
  PadArgs a{};
  int n = 0;
  int64_t most = 0;
  auto one = [&](const void*& p, int64_t& stride, int64_t rows, int64_t cols) {
    if (!fovi::tc_takes(p, stride, 2)) {
      const int64_t pitch = fovi::split_pitch(cols);
      a.t[n++] = PadTask{static_cast<const uint16_t*>(p), stride, reinterpret_cast<uint16_t*>(at), rows, cols, pitch};
      most = std::max(most, rows * pitch / 8);
      p = at;
      stride = pitch;
    }
    at += pad_bytes(rows, cols);
  };
  one(b.x, b.xs, b.M, b.C);
  one(b.wg, b.gs, b.F, b.C);
  one(b.wu, b.us, b.F, b.C);
  one(b.wd, b.ds, b.O, b.F);
  if (g) one(g->dy, g->dys, b.M, b.O);
  pad_kernel<<<dim3((unsigned)std::min<int64_t>((most + 255) / 256, 8 * fovi::sm_count()), n), 256, 0, st>>>(a);
  return fovi::after_launch("pad_kernel");
}

// Rows and channels are counted in 32 bits, twice the hidden channels' bytes too; and a tile's waits are bounded, which its steps of 64 channels have to stay well below.
constexpr int MOST_CHANNELS = 1 << 24;
bool valid(int dtype, int64_t M, int C, int F, int O) {
  return fovi::valid_dtype(dtype) && M >= 0 && M <= (1 << 30) && C >= 1 && C <= MOST_CHANNELS && F >= 1 && F <= MOST_CHANNELS && O >= 1 && O <= MOST_CHANNELS;
}

}  // namespace

extern "C" int64_t fovi_gated_ffn_saved_bytes(int dtype, int64_t tokens, int F) {
  if (!valid(dtype, tokens, 1, F, 1)) return -1;
  return tokens * pitch_of(F) * (dtype == FOVI_BF16 ? 8 : 14);
}

extern "C" int64_t fovi_gated_ffn_workspace_bytes(int dtype, int64_t tokens, int C, int F, int O, int phase) {
  if (!valid(dtype, tokens, C, F, O) || phase < 0 || (phase & 3) > 2 || phase > 6) return -1;
  const bool copies = phase & FOVI_FFN_UNALIGNED;
  phase &= 3;
  Block b{};
  b.M = tokens; b.C = C; b.F = F; b.O = O;
  if (dtype == FOVI_F32 && phase == 0 && fovi::few_float(tokens, C, F, O)) return tokens * pitch_of(F) * 4;
  if (dtype == FOVI_F32) return phase == 1 ? split_backward_at(b, SplitMatrix{}, nullptr).bytes : split_forward_at(b, phase == 2, nullptr).bytes;
  const int64_t extra = copies ? pads_bytes(tokens, C, F, O, phase == 1) : 0;
  if (phase == 1) return extra + back_work(b, pitch_of(F)).bytes;
  if (phase == 0 && fovi::few_block(tokens, C, F, O)) return extra + tokens * pitch_of(F) * 4;
  return extra + (phase == 0 ? padded(tokens * pitch_of(F) * 2) : 0) + fovi::tc_linear_bytes(tokens, O, F, 1);
}

extern "C" int fovi_gated_ffn_forward(const void* x, int dtype, int64_t tokens, int C, int F, int O, int64_t x_stride, const void* gate_weight, int64_t gate_stride,
                                      const void* up_weight, int64_t up_stride, const void* down_weight, int64_t down_stride, const void* gate_bias, const void* up_bias,
                                      const void* down_bias, int activation, void* y, void* saved, void* work, int64_t work_bytes, void* stream) {
  if (!valid(dtype, tokens, C, F, O) || activation < 0 || activation > 1 || x_stride < 0 || gate_stride < 0 || up_stride < 0 || down_stride < 0) return FOVI_ERR_INVALID_ARGUMENT;
  if (tokens == 0) return FOVI_OK;
  if (!x || !gate_weight || !up_weight || !down_weight || !y) return FOVI_ERR_INVALID_ARGUMENT;
  Block b{x, gate_weight, up_weight, down_weight, gate_bias, up_bias, down_bias, tokens, x_stride, gate_stride, up_stride, down_stride, C, F, O, activation};
  const bool copies = dtype == FOVI_BF16 && !boundaries(b, nullptr);
  const int64_t need = fovi_gated_ffn_workspace_bytes(dtype, tokens, C, F, O, (saved ? 2 : 0) | (copies ? FOVI_FFN_UNALIGNED : 0));
  if (work_bytes < need || (need && !work)) return FOVI_ERR_INVALID_ARGUMENT;
  for (const void* p : {(const void*)y, (const void*)work, (const void*)saved})
    if (reinterpret_cast<uintptr_t>(p) % (p == y ? 16 : 32)) return FOVI_ERR_ALIGNMENT;
  auto st = reinterpret_cast<cudaStream_t>(stream);
  char* at = static_cast<char*>(work);
  if (dtype == FOVI_F32) return forward_split(b, y, saved, at, st);
  if (copies) {
    const int rc = pad(b, nullptr, at, st);
    if (rc) return rc;
  }
  const Hidden h = hidden_at(saved ? saved : at, tokens, F, saved != nullptr);
  return forward_bf16(b, y, h, at + (saved ? 0 : padded(tokens * h.pitch * 2)), st);
}

extern "C" int fovi_gated_ffn_backward(const void* x, int dtype, int64_t tokens, int C, int F, int O, int64_t x_stride, const void* gate_weight, int64_t gate_stride,
                                       const void* up_weight, int64_t up_stride, const void* down_weight, int64_t down_stride, int activation, const void* saved,
                                       const void* dy, int64_t dy_stride, void* dx, void* dgate_weight, void* dup_weight, void* ddown_weight, void* dgate_bias,
                                       void* dup_bias, void* ddown_bias, void* work, int64_t work_bytes, void* stream) {
  if (!valid(dtype, tokens, C, F, O) || activation < 0 || activation > 1 || x_stride < 0 || gate_stride < 0 || up_stride < 0 || down_stride < 0 || dy_stride < 0)
    return FOVI_ERR_INVALID_ARGUMENT;
  auto st = reinterpret_cast<cudaStream_t>(stream);
  const size_t size = fovi::dtype_size(dtype);
  if (tokens == 0) {
    const struct { void* p; size_t n; } zero[] = {{dgate_weight, (size_t)F * C}, {dup_weight, (size_t)F * C}, {ddown_weight, (size_t)O * F},
                                                  {dgate_bias, (size_t)F}, {dup_bias, (size_t)F}, {ddown_bias, (size_t)O}};
    for (const auto& z : zero)
      if (z.p) FOVI_CUDA(cudaMemsetAsync(z.p, 0, z.n * size, st));
    return FOVI_OK;
  }
  if (!x || !gate_weight || !up_weight || !down_weight || !saved || !dy || !work) return FOVI_ERR_INVALID_ARGUMENT;
  Block b{x, gate_weight, up_weight, down_weight, nullptr, nullptr, nullptr, tokens, x_stride, gate_stride, up_stride, down_stride, C, F, O, activation};
  Grads g{dy, dy_stride, dx, dgate_weight, dup_weight, ddown_weight, dgate_bias, dup_bias, ddown_bias};
  const bool copies = dtype == FOVI_BF16 && !boundaries(b, &g);
  if (work_bytes < fovi_gated_ffn_workspace_bytes(dtype, tokens, C, F, O, 1 | (copies ? FOVI_FFN_UNALIGNED : 0))) return FOVI_ERR_INVALID_ARGUMENT;
  for (const void* p : {dx, dgate_weight, dup_weight, ddown_weight})
    if (reinterpret_cast<uintptr_t>(p) % 16) return FOVI_ERR_ALIGNMENT;
  if (reinterpret_cast<uintptr_t>(work) % 32 || reinterpret_cast<uintptr_t>(saved) % 32) return FOVI_ERR_ALIGNMENT;
  char* at = static_cast<char*>(work);
  if (dtype == FOVI_F32) return backward_split(b, saved, g, at, st);
  if (copies) {
    const int rc = pad(b, &g, at, st);
    if (rc) return rc;
  }
  return backward_bf16(b, hidden_at(const_cast<void*>(saved), tokens, F, true), g, at, st);
}
