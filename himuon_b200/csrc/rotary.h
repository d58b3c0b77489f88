// Host-side interface of the rotary kernel (rotary_kernels.cu).
#pragma once

#include <cuda_runtime.h>

namespace himuon {

struct RotaryArgs {
  const void* x = nullptr;
  void* y = nullptr;
  const long long* positions = nullptr;          // one for each row; null: row % seq_len
  const unsigned long long* turns = nullptr;     // rotary_dim / 2 frequencies, in 2^-64 turns a position
  long long rows = 0, ld_x = 0, ld_y = 0, seq_len = 1;
  int heads = 0, head_dim = 0, rotary_dim = 0, interleaved = 0, fp32 = 0;
  float cos_factor = 1.f, sin_factor = 1.f;      // of the cosine, and of the sine (its sign turns the rotation around)
};
void rotary(const RotaryArgs& a, cudaStream_t s);

}  // namespace himuon
