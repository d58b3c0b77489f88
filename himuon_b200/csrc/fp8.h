// Host-side interface of the 8-bit kernels (fp8_quantize.cu, fp8_sm100.cu, few_rows_sm100.cu).
#pragma once

#include <cuda_runtime.h>

namespace himuon {

// One 8-bit copy of a matrix: e4m3 values with rows of `ld` bytes, and the scales of blocks of (block_rows, 128).
struct Fp8Out {
  void* values = nullptr;          // null: this copy is not wanted
  float* scales = nullptr;
  long long ld = 0, scale_row = 0, scale_col = 0;      // strides between the scales of neighbouring blocks
  int block_rows = 1;              // 1 or 128
};
// `rows` x `cols` values of bf16 or fp32 as they lie, and turned around.
struct Fp8QuantizeArgs {
  const void* x = nullptr;
  long long rows = 0, cols = 0, ld = 0;
  int fp32 = 0;
  Fp8Out straight, turned;
};
void fp8_quantize(const Fp8QuantizeArgs& a, cudaStream_t s);

struct Fp8Matrix {
  const void* values = nullptr;
  const float* scales = nullptr;
  long long ld = 0, scale_row = 0, scale_col = 0;
  int rows = 0, cols = 0, block_rows = 1;
};
void fp8_dequantize(const Fp8Matrix& m, void* out, long long ld_out, int out_fp32, cudaStream_t s);

// c = a b^T, bf16 or fp32.  a has blocks of 1 or 128 rows, b of 128.  Rows of c are multiples of 16 bytes apart and written in whole groups of 16.
// `powers`: all scales are powers of two (of normal numbers), as fp8_quantize() makes them.  `parts`: fp8_parts_floats() floats of the call's own, for tiles that are
// cut along the inner dimension, whatever the scales are (none are without).
void fp8_product(const Fp8Matrix& a, const Fp8Matrix& b, void* c, long long ld_c, int out_fp32, int powers, float* parts, cudaStream_t s);
long long fp8_parts_floats(const Fp8Matrix& a, const Fp8Matrix& b);
// The same for a few rows of a; c is contiguous.  `early`: b was there before the launch that comes before this one on the stream, and may be read while that still
// runs.  (33 to 64 rows have as many accumulators as a thread has registers: they are the large kernel's.)
// Which of the two: up to 16 rows always; up to 32 of a weight of 16 MB at most, whose time is its launch (24 rows, 2048 -> 2048 7.6 us, 11.7 in the other; 2560 ->
// 9728 17.6 and 14.8, as each of the few products has its scales to load and apply).
constexpr int kFewFp8Rows = 32;
inline bool few_fp8_rows(const Fp8Matrix& a, const Fp8Matrix& b) {
  return a.rows <= kFewFp8Rows / 2 || (a.rows <= kFewFp8Rows && static_cast<long long>(b.rows) * b.cols <= 1LL << 24);
}
void few_rows_fp8_product(const Fp8Matrix& a, const Fp8Matrix& b, void* c, int out_fp32, bool early, cudaStream_t s);

}  // namespace himuon
