// Matrix products of few tokens: what bounds them are the weights' bytes.
#pragma once
#include "product.cuh"

namespace fovi {

// Whether these kernels take a block's forward pass, or an 8-bit product: always for one block of 16 tokens; beyond, the weights come from L2 once for each block of 16, and the tensor
// cores' kernels, which take a fixed time at first, are the faster ones where that is longer.  Both sides measured (us, these / those): block of 96 x 256 channels, 512 and 1024 tokens
// 6.5 / 8.0, 9.9 / 8.0; 384 x 1024, 64, 128 and 192 tokens 6.4 / 10.3, 9.6 / 10.5, 11.6 / 10.5; 768 x 2048, 64 and 96: 13.0 / 14.6, 16.0 / 14.4; 1280 x 1280, 32 and 64: 10.4 / 16.9,
// 14.9 / 14.1; 1280 x 5120, 16 and 32: 14.0 / 19.6, 22.2 / 19.3 (all with h in two parts here, see few_gated).
// 8-bit 384 -> 1024, 64, 96, 128 tokens: 2.5 / 3.9, 3.3 / 4.0, 3.9 / 4.0; 1280 -> 5120, 32, 48: 6.0 / 6.5, 8.0 / 6.6; 5120 -> 1280, 64, 96: 7.5 / 9.0, 9.4 / 9.1.
inline bool few_block(int64_t m, int64_t c, int64_t f, int64_t o) {
  const int64_t channels = c + f < 5000 ? c + f : 5000;
  return m <= 16 || (m <= 1024 && (m + 15) / 16 * f * (2 * c + o) / 3 <= 700000 + 2000 * channels);
}
// A float32 block's, 8 tokens a block, against product_split.cu's: 1280 x 3416, 8 and 16 tokens 47 / 79 and 62 / 80, 32 tokens 118 / 81; 384 x 1024, 32 and 48 tokens 20 / 23 and 25 / 24.
inline bool few_float(int64_t m, int64_t c, int64_t f, int64_t o) { return m <= 16 || (m <= 1024 && (m + 7) / 8 * f * (2 * c + o) / 3 <= 1600000); }
inline bool few_eight(int64_t m, int64_t k, int64_t n) { return m <= 16 || (m <= 1024 && (m + 15) / 16 * n * (k + 1500) <= 10000000 + 7300 * k + 2000 * n); }

// Rows as in TcMatrix: `pitch` values apart, on 16-byte boundaries.
struct FewRows { const void* p; int64_t pitch; };

// h = act(x Wg^T + bg) (x Wu^T + bu) as the sum of two bf16 values, [2][m][pitch]: h rounded to bf16 would put as much into the block's error as its rounded result does, and its rest costs
// few_down no weights.  For up to 16 tokens these bound it (1 x 1280 x 5120: 12.8 us with h in one part, 13.3 in two); beyond, the tokens' loads and products count: 384 x 1024, 64 and 128 tokens 5.5 and 6.4,
// 7.2 and 9.6; 768 x 2048, 64 tokens 9.8 and 13.0; 1280 x 5120, 32 tokens 17.3 and 22.2 (which few_block leaves to the tensor cores' kernels).
int few_gated(const FewRows& x, const FewRows& wg, const FewRows& wu, int m, int n, int k, const void* bg, const void* bu, int act, const FewRows& h, cudaStream_t st);
// y = h W^T + bias, bf16; the launch before it in the stream is few_gated's of the same call.
int few_down(const FewRows& h, const FewRows& w, int m, int n, int k, const void* bias, void* y, cudaStream_t st);
// A float32 block's forward pass, rows of any alignment; h: [m, h_pitch] to work in.
int few_block32(const float* x, int64_t xs, const float* wg, int64_t gs, const float* wu, int64_t us, const float* wd, int64_t ds, int m, int c, int f, int o, const float* bg,
                const float* bu, const float* bd, int act, float* h, int64_t h_pitch, float* y, cudaStream_t st);
// y = scale wscale (q W^T) + bias, y bf16 or float32.
int few_int8(const FewRows& q, const FewRows& w, int m, int n, int k, const float* scale, const float* wscale, const float* bias, void* y, int y_dtype, cudaStream_t st);

}  // namespace fovi
