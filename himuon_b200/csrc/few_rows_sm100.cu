// Products of a few rows (newest tokens) with a large weight, whose bytes are all that counts:  y = x W^T  in bf16, the same of two
// weights with the gated activation between them, and the same in 8 bits with a scale for each block of 128.
//
// A block streams `th` rows of W (of both weights) through a ring of stages in shared memory, 128 bytes of each row and of each row of x a
// stage, by TMA; two blocks to an SM, so that some 190 KB are on the way at any time.  Warps take 16 rows of W each from there: rows of W are the A operand of
// mma.sync, up to 8 rows of x the B operand; 8-bit values go there as fp16 (24 rows of 2560 -> 9728 19.4 us, 21.3 as e4m3).  (tcgen05.mma leaves its sums in tensor
// memory, and blocks with scales of their own would have to be fetched from there one by one; its rate is not needed here.)
//
// A block has as few rows of W as it takes to keep all SMs busy, so that often two or three groups of warps take the stages in turn, and their parts meet in
// shared memory.  Where that would be fewer than 24 rows (a narrow weight, whose inner dimension is long), so that x would be as much to load as W, up to four
// blocks, a cluster, have a part of the inner dimension each, and read one another's parts.  From 33 rows on blocks with 32 rows each have a tile together, which
// takes W from memory once and from the L2 for the others, and has more rows of W for that (64 rows, 2560 x 9728 gated and back: 51 us, 59 in one block with 64
// rows, whose sums fill the registers).  Everything is added up in one order, which goes by the weight's sizes and, from 33 rows on, by the number of such blocks: bits
// repeat, and a row's do not depend on how many rows up to 32 come with it (in 8 bits, up to 16 where the weight is large: more are another kernel's, fp8.h).
//
// A kernel of this kind is over in 8 to 20 us, of which its start is one or two.  So the second of two (the down projection; the product behind a quantisation)
// is launched over the first: it sets up, and fills its ring with W, while that still runs, and waits for it before it asks for x.
//
// What bounds it: memory while the ring is full (6.3 TB/s of W at 24 rows of 2560 x 9728 gated), the start, and the loading warp, whose every instruction costs
// some five cycles: with addresses worked out at each stage it took 500 cycles a stage.  One row, 2048 x 8192 gated and back: 22.5 us for 100.7 MB; 24 rows, 2560 x 9728:
// 36.5 us for 149.4 MB; 8 rows, 2560 -> 9728 in 8 bits with x's quantisation: 12.6 us for 24.9 MB.  Without the clusters and the overlap 30.7, 41.9 and 14.4.
// W loaded from memory straight into the operands' registers took longer (24 rows 38 + 30 us, at that time 22 + 17), so did stages that all warps of a
// block wait for (25 + 47), and loads issued by the group that has emptied a stage (28.8 for 24.4 gated).
#include "activations.cuh"
#include "fp8.h"
#include "gated_mlp.h"
#include "himuon.h"
#include "pair_common.cuh"
#include "sm100_common.cuh"
#include "tma_host.h"

#include <type_traits>

namespace himuon {

namespace {

enum { PLAIN, GATED, EIGHT_BITS };

constexpr int FEW_WARPS = 7, FEW_THREADS = 32 * (1 + FEW_WARPS);      // warp 0: TMA; then 16 rows of W each (with one more, threads would have 96 registers)
constexpr int FEW_ROWS = 16 * FEW_WARPS;
constexpr int FEW_STAGES = 24;
constexpr int FEW_CUT = 4;               // blocks that share a tile, at most
constexpr uint32_t FEW_RING = 96 * 1024;

struct FewDev {
  const float *sx, *sw;                // EIGHT_BITS
  long long sx_row, sx_col, sw_row, sw_col;
  int x_block;
  void *y, *gu;                        // (rows, outer) in bf16 or fp32; GATED: g | u or null (gated_mlp.h)
  uint8_t* gu_low;
  int rows, outer, out_fp32, activation;
  int blocks;                          // of 128 bytes of a row
  int th, tiles, stages;               // rows of W of a tile, tiles of a block, stages of the ring
  int cut;                             // blocks (a cluster) that a tile's inner dimension is dealt out to
  int chunks, x_rows;                  // blocks that have a tile with 32 rows of x each, and rows of x in a load
  int early;                           // W was there before the launch before this one
  int warps, groups;                   // warps that a tile's rows take, and groups of so many, which take stages in turn
  int* status;
};

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Four e4m3 values as fp16, which holds them all.
__device__ __forceinline__ void widen(uint32_t v, uint32_t (&w)[2]) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(w[0]), "=r"(w[1]) : "r"(v));
}
// 32 products of e4m3 values, as two times 16 of fp16: lanes have four neighbouring values along the sum, which may come in any order that is the same in a and b.
__device__ __forceinline__ void mma_e4m3(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  uint32_t w[4][2], v[2][2];
#pragma unroll
  for (int i = 0; i < 4; ++i) widen(a[i], w[i]);
  widen(b0, v[0]);
  widen(b1, v[1]);
  mma_f16(c, w[0][0], w[1][0], w[0][1], w[1][1], v[0][0], v[0][1]);
  mma_f16(c, w[2][0], w[3][0], w[2][1], w[3][1], v[1][0], v[1][1]);
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&v)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ld_cluster(uint32_t addr, float (&v)[1]) { asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v[0]) : "r"(addr) : "memory"); }
__device__ __forceinline__ void ld_cluster(uint32_t addr, float (&v)[4]) {
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void expect(uint32_t bar, uint32_t bytes, uint32_t e) {
  asm volatile("{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %2, 0;\n\t@e mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(bar), "r"(bytes), "r"(e) : "memory");
}
__device__ __forceinline__ void load(uint32_t dst, const CUtensorMap* tm, uint32_t bar, int x, int y, uint32_t e) {
  asm volatile(
      "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %5, 0;\n\t"
      "@e cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n\t}" ::"r"(dst), "l"(tm), "r"(bar), "r"(x), "r"(y), "r"(e)
      : "memory");
}
// 16 bytes of a row of 128, where the swizzle has put them.
__device__ __forceinline__ uint32_t cell(uint32_t base, int row, int chunk) { return base + row * 128 + ((chunk ^ (row & 7)) << 4); }

__device__ __forceinline__ float activate_any(int activation, float g) {
  return activation == kSilu ? activate<kSilu>(g) : activation == kGelu ? activate<kGelu>(g) : activation == kGeluTanh ? activate<kGeluTanh>(g) : activate<kRelu>(g);
}
// The result of one row of W (of both) and one of x.
template <int KIND>
__device__ __forceinline__ void put_result(const FewDev& p, int feature, int row, float v, float u) {
  if (feature >= p.outer) return;
  const long long at = static_cast<long long>(row) * p.outer + feature;
  if constexpr (KIND == GATED) {
    reinterpret_cast<__nv_bfloat16*>(p.y)[at] = __float2bfloat16_rn(activate_any(p.activation, v) * u);
    if (p.gu) {
      uint16_t* gu = static_cast<uint16_t*>(p.gu) + 2LL * row * p.outer + feature;
      uint8_t* low = p.gu_low + 2LL * row * gated_low(p.outer) + feature;
      gu[0] = static_cast<uint16_t>(__float_as_uint(v) >> 16);
      gu[p.outer] = static_cast<uint16_t>(__float_as_uint(u) >> 16);
      low[0] = static_cast<uint8_t>(__float_as_uint(v) >> 8);
      low[gated_low(p.outer)] = static_cast<uint8_t>(__float_as_uint(u) >> 8);
    }
  } else if (p.out_fp32) {
    reinterpret_cast<float*>(p.y)[at] = v;
  } else {
    reinterpret_cast<__nv_bfloat16*>(p.y)[at] = __float2bfloat16_rn(v);
  }
}

struct FewBars {
  uint64_t full[FEW_STAGES], empty[FEW_STAGES];
  int abort_flag;
};

// NT: groups of eight rows of x.
template <int KIND, int NT>
__global__ void __launch_bounds__(FEW_THREADS, 2)
few_rows_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW0, const __grid_constant__ CUtensorMap tmW1, FewDev p) {
  constexpr int MATS = KIND == GATED ? 2 : 1, NX = NT * 8;
  constexpr int PER_SUB = KIND == EIGHT_BITS ? 128 : 64;        // values in 128 bytes
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_up_1024(smem_raw);
  FewBars* bars = reinterpret_cast<FewBars*>(smem + FEW_RING);
  volatile int* abort_flag = &bars->abort_flag;
  const bool joined = p.groups > 1 || p.cut > 1;
  const int line = p.warps * 16 + 4;                   // of parts: a row of x by all rows of W (4 more, so that a warp's values lie in 32 banks)
  const int warp = warp_id(), lane = threadIdx.x & 31;
  const int of = static_cast<int>(blockIdx.x) / p.cut, rank = static_cast<int>(blockIdx.x) - of * p.cut, first = of / p.chunks * p.th * p.tiles;
  const int row0 = of % p.chunks * 32, rows = min(p.rows - row0, 32);
  const int kb0 = p.blocks * rank / p.cut, kb1 = p.blocks * (rank + 1) / p.cut;
  const uint32_t w_bytes = static_cast<uint32_t>(p.th) * 128, stage_bytes = MATS * w_bytes + NX * 128;
  if (KIND == GATED) launch_dependents();              // (the down projection, whose W is not made here; nothing is launched over one that was launched so itself)
  if (static_cast<int>(threadIdx.x) < p.stages) { mbar_init(&bars->full[threadIdx.x], 1); mbar_init(&bars->empty[threadIdx.x], p.warps); }
  if (threadIdx.x == 0) bars->abort_flag = 0;
  if (warp == 0) mbar_fence_init();
  __syncthreads();

  if (warp == 0) {
    // (a stage costs its bytes' time or this loop's instructions, which take some five cycles each: addresses go along, nothing is worked out anew)
    const uint32_t e = elect_one(), bytes = MATS * w_bytes + p.x_rows * 128, ring = smem_u32(smem), full0 = smem_u32(bars->full);
    const int n = kb1 - kb0, ahead = p.early ? min(p.stages, n) : 0;
    for (int i = 0; i < ahead; ++i) {                    // W while the kernel before may still be writing x
      expect(full0 + i * 8, bytes, e);
      load(ring + i * stage_bytes, &tmW0, full0 + i * 8, (kb0 + i) * PER_SUB, first, e);
      if (MATS == 2) load(ring + i * stage_bytes + w_bytes, &tmW1, full0 + i * 8, (kb0 + i) * PER_SUB, first, e);
    }
    wait_for_previous();
    for (int i = 0; i < ahead; ++i) load(ring + i * stage_bytes + MATS * w_bytes, &tmX, full0 + i * 8, (kb0 + i) * PER_SUB, row0, e);
    int stage = ahead;
    uint32_t phase = 1, at = ring + ahead * stage_bytes, bar = full0 + ahead * 8;
    bool ok = true;
    for (int tile = 0, f0 = first; ok && tile < p.tiles && f0 < p.outer; ++tile, f0 += p.th) {
      int k = (kb0 + (tile == 0 ? ahead : 0)) * PER_SUB;
#pragma unroll 1
      for (int left = n - (tile == 0 ? ahead : 0); left > 0; --left, k += PER_SUB) {      // (behind the last value: zeros)
        if (stage == p.stages) { stage = 0; phase ^= 1; at = ring; bar = full0; }
        if (!mbar_wait_warp(&bars->empty[stage], phase, abort_flag, p.status, 1)) { ok = false; break; }
        expect(bar, bytes, e);
        load(at, &tmW0, bar, k, f0, e);
        if (MATS == 2) load(at + w_bytes, &tmW1, bar, k, f0, e);
        load(at + MATS * w_bytes, &tmX, bar, k, row0, e);
        ++stage;
        at += stage_bytes;
        bar += 8;
      }
    }
  } else {
    const int group = (warp - 1) / p.warps, m0 = (warp - 1 - group * p.warps) * 16, r = lane >> 2, t = lane & 3;
    const uint32_t ring = smem_u32(smem);
    // the lane's addresses of ldmatrix: rows 0-7 and 8-15 of W by bytes 0-15 and 16-31; eight rows of x by four times 16 bytes
    const int a_row = m0 + (lane & 15), a_chunk = lane >> 4, b_row = lane & 7, b_chunk = lane >> 3;
    int stage = group;                                   // (groups take turns; stages are a multiple of them)
    uint32_t phase = 0;
    bool ok = group < p.groups;
    if (KIND == EIGHT_BITS) wait_for_previous();         // (scales of x)
    for (int tile = 0; tile < p.tiles && first + tile * p.th < p.outer; ++tile) {
      const int f0 = first + tile * p.th;
      float acc[MATS][NT][4] = {};
      const float *sw0 = nullptr, *sw1 = nullptr;
      float by_w[2] = {}, by_x[NT][2] = {}, next_w[2] = {}, next_x[NT][2] = {};
      const bool x_blocks = p.x_block > 1;                 // (of 128 rows: the first has them all)
      auto load_scales = [&](int block) {
        const int at = min(block, p.blocks - 1);
        next_w[0] = __ldg(sw0 + at * p.sw_col);
        next_w[1] = __ldg(sw1 + at * p.sw_col);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) next_x[n][j] = __ldg(p.sx + (x_blocks ? 0 : min(n * 8 + 2 * t + j, p.rows - 1)) * p.sx_row + at * p.sx_col);
      };
      if constexpr (KIND == EIGHT_BITS) {
        sw0 = p.sw + static_cast<long long>(min(f0 + m0 + r, p.outer - 1) / 128) * p.sw_row;
        sw1 = p.sw + static_cast<long long>(min(f0 + m0 + r + 8, p.outer - 1) / 128) * p.sw_row;
        load_scales(kb0 + group);
      }
      for (int kb = kb0 + group; ok && kb < kb1; kb += p.groups) {
        if constexpr (KIND == EIGHT_BITS) {                  // (those of a turn are on their way during the one before)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            by_w[j] = next_w[j];
#pragma unroll
            for (int n = 0; n < NT; ++n) by_x[n][j] = next_x[n][j];
          }
          load_scales(kb + p.groups);
        }
        if (!mbar_wait_warp(&bars->full[stage], phase, abort_flag, p.status, 3)) { ok = false; break; }
        const uint32_t base = ring + stage * stage_bytes, x_base = base + MATS * w_bytes;
        // A turn is latency: as many operands as there are registers for are asked for before the first product.  In 8 bits every other product goes to another
        // sum, and the two are scaled and added one after the other: with many rows there are registers for one of them at a time, and the order is the same.
        constexpr int HALVES = NT <= 2 ? 2 : 1, STEPS = 2 * HALVES;
        constexpr bool ONE_SUM = KIND == EIGHT_BITS && HALVES == 1;
        // products 2 half and 2 half + 1 of the four, or (ONE_SUM) half and half + 2
        const int b_at = ONE_SUM ? (b_chunk & 1) + (b_chunk >> 1) * 4 : b_chunk;
        constexpr int B_HALF = ONE_SUM ? 2 : 4, A_STEP = ONE_SUM ? 4 : 2, A_HALF = ONE_SUM ? 2 : 4;
#pragma unroll 1
        for (int half = 0; half < 2; half += HALVES) {
          float c[HALVES][NT][4] = {};
          uint32_t b[HALVES][NT][4];
#pragma unroll
          for (int h = 0; h < HALVES; ++h)
#pragma unroll
            for (int n = 0; n < NT; ++n) ldmatrix4(b[h][n], cell(x_base, n * 8 + b_row, (half + h) * B_HALF + b_at));
          uint32_t a[STEPS][MATS][4];
#pragma unroll
          for (int m = 0; m < MATS; ++m)
#pragma unroll
            for (int k = 0; k < STEPS; ++k) ldmatrix4(a[k][m], cell(base + m * w_bytes, a_row, half * A_HALF + k * A_STEP + a_chunk));
#pragma unroll
          for (int k = 0; k < STEPS; ++k)
#pragma unroll
            for (int m = 0; m < MATS; ++m)
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                const uint32_t b0 = b[k / 2][n][2 * (k % 2)], b1 = b[k / 2][n][2 * (k % 2) + 1];
                if constexpr (KIND == EIGHT_BITS) mma_e4m3(c[k % HALVES][n], a[k][m], b0, b1);
                else mma_bf16(acc[m][n], a[k][m], b0, b1);
              }
          if constexpr (KIND == EIGHT_BITS) {
#pragma unroll
            for (int h = 0; h < HALVES; ++h)
#pragma unroll
              for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[0][n][j] = fmaf(c[h][n][j], by_w[j >> 1] * by_x[n][j & 1], acc[0][n][j]);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->empty[stage]);
        stage += p.groups;
        if (stage >= p.stages) { stage -= p.stages; phase ^= 1; }
      }
      if (!joined) {                                     // (one group: it has them all)
        if (ok) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int f = m0 + r + 8 * (j >> 1);
              if (f < p.th && n * 8 + 2 * t + (j & 1) < rows) put_result<KIND>(p, f0 + f, row0 + n * 8 + 2 * t + (j & 1), acc[0][n][j], acc[MATS - 1][n][j]);
            }
        }
      } else {                                           // (one tile: the ring has been read to its end by all warps that the barrier waits for)
        named_barrier(1, 32 * FEW_WARPS);
        if (group < p.groups) {
          float* s_part = reinterpret_cast<float*>(smem) + group * MATS * NX * line;
#pragma unroll
          for (int m = 0; m < MATS; ++m)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int j = 0; j < 4; ++j) s_part[(m * NX + n * 8 + 2 * t + (j & 1)) * line + m0 + r + 8 * (j >> 1)] = acc[m][n][j];
        }
      }
      if (!ok && group < p.groups) break;
    }
  }
  if (!joined) return;
  // the groups' parts, of all blocks of the cluster, neighbouring features next to one another; the blocks share the results
  __syncwarp();
  if (p.cut > 1) cluster_sync_all();
  else __syncthreads();
  const uint32_t parts = smem_u32(smem), step = MATS * NX * line * 4, of_w1 = (MATS - 1) * NX * line * 4;
  // V neighbouring features a thread: four where that leaves one for each thread (24 rows of 40 features: 1.2 us for 2.4 one by one), else one
  auto join = [&](auto width) {
    constexpr int V = decltype(width)::value;
    const int line_of = p.th / V, out = line_of * rows;
    for (int o = rank * FEW_THREADS + static_cast<int>(threadIdx.x); o < out; o += p.cut * FEW_THREADS) {
      const int row = o / line_of, f = (o - row * line_of) * V;
      float v[MATS][V] = {};
      const uint32_t at = parts + (row * line + f) * 4;
      for (int g = 0; g < p.groups; ++g)
#pragma unroll
        for (int m = 0; m < MATS; ++m) {
          float u[FEW_CUT][V];
#pragma unroll
          for (int c = 0; c < FEW_CUT; ++c)
            if (c < p.cut) ld_cluster((p.cut > 1 ? map_to_cta(at, c) : at) + g * step + m * of_w1, u[c]);
#pragma unroll
          for (int c = 0; c < FEW_CUT; ++c)
            if (c < p.cut)
#pragma unroll
              for (int i = 0; i < V; ++i) v[m][i] += u[c][i];
        }
#pragma unroll
      for (int i = 0; i < V; ++i) put_result<KIND>(p, first + f + i, row0 + row, v[0][i], v[MATS - 1][i]);
    }
  };
  if (p.th * rows >= 2 * FEW_THREADS * p.cut) join(std::integral_constant<int, 4>{});
  else join(std::integral_constant<int, 1>{});
  __syncwarp();
  if (p.cut > 1) cluster_sync_all();   // (nobody leaves while others read its parts)
}

struct FewOperands {
  const void *x = nullptr, *w0 = nullptr, *w1 = nullptr;
  long long ld_x = 0, ld_w0 = 0, ld_w1 = 0;              // bytes between rows
  int inner = 0, esz = 2;                                // values of a row and their bytes
};
CUtensorMap few_map(const void* ptr, int rows, const FewOperands& o, long long ld, int box_rows) {
  const uint64_t dims[2] = {static_cast<uint64_t>(o.inner), static_cast<uint64_t>(rows)}, strides[1] = {static_cast<uint64_t>(ld)};
  const uint32_t box[2] = {static_cast<uint32_t>(128 / o.esz), static_cast<uint32_t>(box_rows)};
  return make_tmap(ptr, 2, dims, strides, box, o.esz, true);
}

template <int KIND, int NT>
void launch(const FewOperands& o, FewDev p, cudaStream_t s) {
  constexpr int MATS = KIND == GATED ? 2 : 1, NX = NT * 8;
  constexpr size_t SMEM = 1024 + FEW_RING + sizeof(FewBars);
  static_assert(2 * SMEM <= 232448 && MATS * NX * (FEW_ROWS + 4 * FEW_WARPS) * sizeof(float) <= FEW_RING &&
                    (MATS * FEW_ROWS + 32) * 128 <= FEW_RING, "shared memory of two blocks exceeded");
  const auto kernel = few_rows_kernel<KIND, NT>;
  p.blocks = (o.inner * o.esz + 127) / 128;
  // Rows of W in equal shares over two blocks a SM, in tiles of up to FEW_ROWS.
  // Where that leaves a block fewer than 24 rows, so that up to 32 of x would be as much to load as W, blocks share tiles instead.
  p.chunks = (p.rows + 31) / 32;
  p.x_rows = p.rows < 32 ? p.rows : 32;
  const int slots = 2 * num_sms() / p.chunks;
  p.cut = 1;
  while (p.cut < FEW_CUT && static_cast<long long>(p.outer) * p.cut < 24LL * slots && p.blocks >= 32 * p.cut) p.cut *= 2;
  const int share = static_cast<int>((static_cast<long long>(p.outer) * p.cut + slots - 1) / slots + 7) / 8 * 8;
  p.tiles = (share + FEW_ROWS - 1) / FEW_ROWS;
  p.th = ((share + p.tiles - 1) / p.tiles + 7) / 8 * 8;
  p.warps = (p.th + 15) / 16;
  // Bytes of a stage and groups go by the weight alone (with the most rows of x that there may be), since what a group has, and with it the order of sums, does.
  const int weight = MATS * p.th * 128;
  const int least = static_cast<int>(FEW_RING) / (weight + 32 * 128);
  p.groups = p.tiles > 1 ? 1 : FEW_WARPS / p.warps < least ? FEW_WARPS / p.warps : least;
  const int sub_bytes = weight + NX * 128;
  const int fit = static_cast<int>(FEW_RING) / sub_bytes;
  p.stages = fit < FEW_STAGES ? fit : FEW_STAGES;
  // (A stage is always the same group's: a group that met another's could be a whole round ahead of it, where a barrier's phases look alike.)
  p.stages -= p.stages % p.groups;
  p.status = status_word_ptr();
  const long long group = static_cast<long long>(p.th) * p.tiles, grid = (p.outer + group - 1) / group * p.chunks * p.cut;
  const CUtensorMap tx = few_map(o.x, p.rows, o, o.ld_x, p.x_rows), t0 = few_map(o.w0, p.outer, o, o.ld_w0, p.th), t1 = MATS == 2 ? few_map(o.w1, p.outer, o, o.ld_w1, p.th) : t0;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(SMEM));
  if (e == cudaSuccess) {
    cudaLaunchAttribute attrs[2];
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(grid));
    cfg.blockDim = dim3(FEW_THREADS);
    cfg.dynamicSmemBytes = SMEM;
    cfg.stream = s;
    cfg.attrs = attrs;
    if (p.early) {
      attrs[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      attrs[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (p.cut > 1) {
      attrs[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
      attrs[cfg.numAttrs].val.clusterDim.x = static_cast<unsigned>(p.cut);
      attrs[cfg.numAttrs].val.clusterDim.y = attrs[cfg.numAttrs].val.clusterDim.z = 1;
      ++cfg.numAttrs;
    }
    e = cudaLaunchKernelEx(&cfg, kernel, tx, t0, t1, p);
  }
  if (e != cudaSuccess) throw std::runtime_error(std::string("himuon product of few rows: launch failed: ") + cudaGetErrorString(e));
}
template <int KIND>
void launch_rows(const FewOperands& o, const FewDev& p, cudaStream_t s) {
  if (p.rows <= 0 || p.rows > (KIND == EIGHT_BITS ? kFewFp8Rows : kFewProductRows) || p.outer <= 0 || o.inner <= 0) throw std::runtime_error("himuon product of few rows: bad sizes");
  if (p.rows <= 8) launch<KIND, 1>(o, p, s);
  else if (p.rows <= 16) launch<KIND, 2>(o, p, s);
  else launch<KIND, 4>(o, p, s);
}

}  // namespace

void few_rows_product(const void* x, long long ld_x, const void* w, long long ld_w, void* y, int rows, int inner, int outer, bool early, cudaStream_t s) {
  FewOperands o;
  o.x = x; o.ld_x = 2 * ld_x; o.w0 = w; o.ld_w0 = 2 * ld_w; o.inner = inner;
  FewDev p{};
  p.y = y; p.rows = rows; p.outer = outer; p.early = early;
  launch_rows<PLAIN>(o, p, s);
}

void few_rows_gated_up(const GatedUpArgs& a, cudaStream_t s) {
  FewOperands o;
  o.x = a.x; o.ld_x = 2 * a.ld_x; o.w0 = a.wg; o.ld_w0 = 2 * a.ld_wg; o.w1 = a.wu; o.ld_w1 = 2 * a.ld_wu; o.inner = a.hidden;
  FewDev p{};
  p.y = a.h; p.gu = a.gu; p.gu_low = static_cast<uint8_t*>(a.gu_low);
  p.rows = a.rows; p.outer = a.inter; p.activation = a.activation;
  if (a.activation < kSilu || a.activation > kRelu) throw std::runtime_error("himuon gated_mlp: unknown activation");
  launch_rows<GATED>(o, p, s);
}

void few_rows_fp8_product(const Fp8Matrix& a, const Fp8Matrix& b, void* c, int out_fp32, bool early, cudaStream_t s) {
  if (a.cols != b.cols || b.block_rows != 128) throw std::runtime_error("himuon fp8_product: bad sizes");
  FewOperands o;
  o.x = a.values; o.ld_x = a.ld; o.w0 = b.values; o.ld_w0 = b.ld; o.inner = a.cols; o.esz = 1;
  FewDev p{};
  p.sx = a.scales; p.sx_row = a.scale_row; p.sx_col = a.scale_col; p.x_block = a.block_rows;
  p.sw = b.scales; p.sw_row = b.scale_row; p.sw_col = b.scale_col;
  p.y = c; p.out_fp32 = out_fp32; p.early = early;
  p.rows = a.rows; p.outer = b.rows;
  launch_rows<EIGHT_BITS>(o, p, s);
}

}  // namespace himuon
