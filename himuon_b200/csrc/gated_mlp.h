// Host-side interface of the gated feed-forward kernels (gated_mlp_sm100.cu, few_rows_sm100.cu).
#pragma once

#include <cuda_runtime.h>

namespace himuon {

enum Activation { kSilu = 0, kGelu = 1, kGeluTanh = 2, kRelu = 3 };

// What the backward pass needs of g = x wg^T and u = x wu^T: their upper 16 bits (truncated, unlike bf16), (rows, 2 * inter), and the 8 below,
// (rows, 2 * gated_low(inter)).  So they are off by at most 2^-15 of themselves, for half as many bytes again; kept in bf16 alone they would be off by as much
// as what is made of them is rounded, and the gradients of both weights by 3.0e-3 instead of 2.4e-3.
constexpr int gated_low(int inter) { return (inter + 15) / 16 * 16; }

// h = act(x wg^T) * (x wu^T), all bf16 with rows on 16-byte boundaries.  With `gu` and `gu_low`: g and u too.
struct GatedUpArgs {
  const void *x = nullptr, *wg = nullptr, *wu = nullptr;
  void *h = nullptr, *gu = nullptr, *gu_low = nullptr;
  long long ld_x = 0, ld_wg = 0, ld_wu = 0;      // (h and gu are contiguous)
  int rows = 0, hidden = 0, inter = 0, activation = 0;
};
void gated_up(const GatedUpArgs& a, cudaStream_t s);

// dgu = (dh * u * act'(g) | dh * act(g)) with dh = dy wd, which stays on the chip; wd is (hidden, inter).
struct GatedDownGradArgs {
  const void *dy = nullptr, *wd = nullptr, *gu = nullptr, *gu_low = nullptr;
  void* dgu = nullptr;
  long long ld_dy = 0, ld_wd = 0;
  int rows = 0, hidden = 0, inter = 0, activation = 0;
};
void gated_down_grad(const GatedDownGradArgs& a, cudaStream_t s);

// Products with a few rows (up to kFewProductRows), whose weight is all that counts: y = x w^T in bf16, or gated_up().
// `early`: w was there before the launch that comes before this one on the stream, and may be read while that still runs.
constexpr int kFewProductRows = 384;
// Whether the gated block takes them: up to 32 rows always, up to 64 unless the weights are large (64 rows of 2048 x 6144, gated and back: 29 us, 31 in tiles of all rows,
// of 2560 x 9728 51 and 45), and up to 384 of small ones (128 rows of 640 x 1728 13 and 19, of 1360 x 2472 22 and 31, 384 of 640 x 1728 18 and 19; but 192 of 472 x 5648 33 and 24).
inline bool few_gated_rows(long long rows, long long hidden, long long inter) {
  return rows <= 32 || (rows <= 64 && hidden * inter <= 1LL << 24) || (rows <= kFewProductRows && rows * hidden * inter <= 400000000);
}
void few_rows_product(const void* x, long long ld_x, const void* w, long long ld_w, void* y, int rows, int inner, int outer, bool early, cudaStream_t s);
void few_rows_gated_up(const GatedUpArgs& a, cudaStream_t s);

}  // namespace himuon
