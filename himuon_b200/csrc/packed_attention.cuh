// What the forward and the backward kernels of packed attention share (packed_attention_sm100.cu has the formulas and the tiles).
#pragma once

#include <atomic>
#include <string>
#include <type_traits>

#include "attention_common.cuh"

namespace himuon {


struct PackedDev {
  const PackedTile* tiles;
  void* o; float* nlse; float* ndelta;               // minus the base-2 log-sum-exp of the scaled scores, minus delta
  const void* o_in; const void* d_o;
  signed char* o_low;                                // (Hq, tiles, low_ld / 16, 128, 16)
  int low_ld;
  void* dq; void* dk; void* dv;
  int Hq, Hkv, hd;
  int tokens, rows;                                  // rows from `tokens` on belong to no document
  int n_items;
  int pair_heads;                                    // forward: 1 where an item is one tile of two heads
  int split_heads;                                   // dK / dV: 1 where an item is one query head's part of them
  float* dk_part; float* dv_part;                    // (Hq, stat_rows, hd) each
  long long stat_rows;                               // rows of statistics per head: 128 for each tile
  long long ld_o, ld_do, ld_dq, ld_dk, ld_dv;
  float scale_log2, scale;
  int* status;
};

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Rows from `row0` to `rows` of a swizzled tile (halves `half` bytes apart) set to zero by a warp, ahead of a product that it issues.
template <int NH>
__device__ __forceinline__ void clear_rows(uint8_t* tile, uint32_t half, int row0, int rows, int lane) {
  const int n = (rows - row0) * 8;                   // 16-byte pieces of a half
#pragma unroll
  for (int j = 0; j < NH; ++j)
    for (int i = lane; i < n; i += 32) *reinterpret_cast<uint4*>(tile + j * half + row0 * 128 + i * 16) = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  __syncwarp();
}

// delta is a difference's second half: for a row whose softmax has one weight near 1, dP - delta is small beside either, and O in bf16 would leave it
// half a bit of its 8 in error.  So the forward pass of training keeps 8 bits more: what O's fp32 word has above (or lacks) of the word of its
// bf16, in units of 2^-8 of its last place.  low_of packs four of them, with_low adds one to its bf16.
__device__ __forceinline__ uint32_t low_of(float f0, float f1, float f2, float f3, uint32_t b01, uint32_t b23) {
  // (half a place up, rounded down to even, is 128 units, which are one too many)
  const int d0 = min(__float_as_int(f0) - static_cast<int>(b01 << 16) + 0x80, 0x7FFF), d1 = min(__float_as_int(f1) - static_cast<int>(b01 & 0xFFFF0000u) + 0x80, 0x7FFF);
  const int d2 = min(__float_as_int(f2) - static_cast<int>(b23 << 16) + 0x80, 0x7FFF), d3 = min(__float_as_int(f3) - static_cast<int>(b23 & 0xFFFF0000u) + 0x80, 0x7FFF);
  return __byte_perm(__byte_perm(d0, d1, 0x0051), __byte_perm(d2, d3, 0x0051), 0x5410);
}
template <int I>
__device__ __forceinline__ float with_low(uint32_t bf16_word, uint32_t low) {     // bf16_word: a bf16 as the upper half, zeros below
  uint32_t d;                                        // 0, the byte, and twice its sign
  asm("prmt.b32 %0, %1, 0, %2;" : "=r"(d) : "r"(low), "n"(0x0004 | I << 4 | (8 | I) << 8 | (8 | I) << 12));
  return __uint_as_float(bf16_word + d);
}

// Where a tile's low bits of a column are: 16 columns of all its rows together, which the threads of the forward pass, one row each, store
// without gaps (24 documents, 8192 tokens, 16 heads over 8: 62 us against 63 with a row's bytes in one piece).
__device__ __forceinline__ long long low_at(const PackedDev& p, int head, int slot, int row, int col) {
  return (head * p.stat_rows + static_cast<long long>(slot) * AT) * p.low_ld + ((col >> 4) * AT + row) * 16 + (col & 15);
}

// Rows that belong to no document, zeroed by the threads of all blocks.
__device__ __forceinline__ void zero_padding(void* out, long long ld, int from, int to, int cols, int thread, int threads) {
  const int per_row = cols / 8;
  const long long n = static_cast<long long>(to - from) * per_row;
  for (long long i = static_cast<long long>(blockIdx.x) * threads + thread; i < n; i += static_cast<long long>(gridDim.x) * threads)
    *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(out) + (from + i / per_row) * ld + (i % per_row) * 8) = make_uint4(0, 0, 0, 0);
}
// The same in the uniform registers of a converged warp.  (What comes from memory is not uniform to the compiler, nor is anything in a
// loop that it bounds: every operand of every MMA would be moved there.)
__device__ __forceinline__ int uniform(int x) { return static_cast<int>(__reduce_or_sync(0xffffffffu, static_cast<uint32_t>(x))); }
// Items are listed by falling work; the blocks take them in turns, back and forth.
__device__ __forceinline__ int my_turn(int round) {
  const int g = static_cast<int>(gridDim.x), b = static_cast<int>(blockIdx.x);
  return round * g + ((round & 1) ? g - 1 - b : b);
}
__device__ __forceinline__ void tma_store_4d(const CUtensorMap* tmap, const void* smem_src, int x, int y, int z, int w, uint32_t e) {
  asm volatile("{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %6, 0;\n\t"
               "@e cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];\n\t}"
               ::"l"(tmap), "r"(smem_u32(smem_src)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(e)
               : "memory");
}
// Whether the phase is over, without a wait; the same in all lanes.
__device__ __forceinline__ bool mbar_peek(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return __all_sync(0xffffffffu, ok != 0);
}

// ---------------------------------------------------------------- host
inline void check_packed(const PackedAttnArgs& a) {
  if (a.Hq <= 0 || a.Hkv <= 0 || a.Hq % a.Hkv || a.rows <= 0 || a.n_tiles < 0) throw std::runtime_error("himuon packed attention: bad sizes");
  if (a.hd <= 0 || a.hd > 128 || a.hd % 8) throw std::runtime_error("himuon packed attention: head_dim must be a multiple of 8 up to 128");
  // (blocks look two turns past the last item, in 32 bits: my_turn)
  if (static_cast<long long>(a.n_tiles) * a.Hq >= (1LL << 31) - (1 << 16)) throw std::runtime_error("himuon packed attention: too many tiles for one launch");
}
inline PackedDev make_dev(const PackedAttnArgs& a) {
  PackedDev p{};
  p.o = a.o; p.o_in = a.o; p.d_o = a.d_o; p.nlse = a.lse; p.ndelta = a.delta; p.dq = a.dq; p.dk = a.dk; p.dv = a.dv;
  p.o_low = a.o_low; p.low_ld = (a.hd + 15) / 16 * 16;
  p.Hq = a.Hq; p.Hkv = a.Hkv; p.hd = a.hd; p.tokens = a.tokens; p.rows = a.rows;
  p.stat_rows = static_cast<long long>(a.n_tiles) * AT;
  p.ld_o = a.ld_o; p.ld_do = a.ld_do; p.ld_dq = a.ld_dq; p.ld_dk = a.ld_dk; p.ld_dv = a.ld_dv;
  p.scale = a.scale; p.scale_log2 = a.scale * kLog2e;
  p.status = status_word_ptr();
  return p;
}
// Once for each kernel and device.
template <typename K>
void allow_smem(K kern, size_t bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (bit && (done.load(std::memory_order_relaxed) & bit)) return;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  if (e != cudaSuccess) throw std::runtime_error(std::string("himuon packed attention: ") + cudaGetErrorString(e));
  done.fetch_or(bit, std::memory_order_relaxed);
}
inline void check_packed_launch(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) throw std::runtime_error(std::string("himuon packed attention ") + what + " launch failed: " + cudaGetErrorString(e));
}

}  // namespace himuon
