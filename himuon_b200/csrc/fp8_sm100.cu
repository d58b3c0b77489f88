// Product of two 8-bit matrices with a scale for each block of 128:  c_ij = sum over blocks b of  sa_i,b * sb_j,b * (sum of the block's qa_ik qb_jk).
// A CTA pair has 256 x 256 of c (gemm2_sm100.cu has the protocol of pairs); a block of 256 x 256 x 128 takes its tensor cores 512 cycles, in which
// each CTA loads 32 KB.  With one CTA to a tile of 128 x 256 it would be 48 KB in the same time, more than an SM takes in.  Two kernels:
//
// Scales that are powers of two (what fp8_quantize() makes) go to the tensor core: its block-scaled form multiplies each 32 products by two such
// scales, which it takes from tensor memory, eight bits of exponent each, four blocks in a word.  c stays in tensor memory for the whole inner dimension.
// Four warps keep the scales coming.  There is room for one accumulator beside them, so the eight warps of the epilogue take all of it into registers, give it back,
// and round and store while the next tile is under way.  8192 x 9728 x 2560 156 us, 8192 x 2560 x 9728 154 (2.6 to 2.7 PFLOP/s); the issuing warp's own
// instructions are what bounds it, some 70 cycles a product and a few hundred around a stage (stages of one block 185 us).
//
// Other scales: the tensor core sums the 128 products of a block, and each block's sums are read from tensor memory, scaled and added up in registers, in
// fp32.  As b has blocks of 128 rows, a thread, which has one row of a and 128 columns, needs one factor a block.  Two accumulators, so that one block is added
// up beside the products of the next.  210 and 212 us: it takes the hand-on of a block between the tensor core and both CTAs' warps, there and back, for each 512
// cycles of products (187 us with nothing but the hand-on).  Commits of their own for the producer and for the sums 219; sixteen warps with 64 columns each 302 for
// 262, at an earlier state; columns on their way while others are added up, no difference.
#include "fp8.h"
#include "gemm_epilogue.cuh"
#include "himuon.h"
#include "kernel_host.h"
#include "pair_common.cuh"
#include "sm100_common.cuh"
#include "tma_host.h"

#include <atomic>
#include <type_traits>

namespace himuon {

namespace {

constexpr int F8_THREADS = 384;      // warps 0-3: TMA, MMA, none, none; 4-11: sums, two groups of four
// Registers of a thread at launch, and after the first four warps have given some to the others, whose sums take 128.
constexpr int F8_REGS = 168, F8_REGS_FEW = 104, F8_REGS_SUMS = 200;
static_assert(F8_REGS_FEW + 2 * F8_REGS_SUMS <= 3 * F8_REGS, "more registers than the block was launched with");
constexpr int F8_STAGES = 6;
constexpr int F8_BAND = 8;           // rows of tiles in a band (tile_at)
constexpr int F8_K = 128;            // values of a block, a 128-byte row of shared memory
constexpr uint32_t F8_A = BM * F8_K, F8_STAGE = 2 * F8_A;

struct Fp8Dev {
  const float *sa, *sb;
  long long sa_row, sa_col, sb_row, sb_col;
  int a_block;                       // rows of a block of a
  int rows, cols, tiles_m, tiles_n, kblocks, band;
  int whole, items, cuts;            // tiles that are taken whole, and each of the others in so many parts along the inner dimension
  int* status;
};

__device__ __forceinline__ void umma2_f8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate, uint32_t e) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(e)
      : "memory");
}
// Tiles in the order in which they are taken: by bands of `band` rows of tiles, down and then along, so that the tiles under way share rows of both operands.
__device__ __forceinline__ void tile_at(const Fp8Dev& p, int tile, int& mt, int& nt) {
  const int per = p.band * p.tiles_n, b = tile / per, at = tile - b * per, first = b * p.band, size = min(p.tiles_m - first, p.band);
  nt = at / size;
  mt = first + at - nt * size;
}
// One of the `items`: blocks kb0 to kb1 - 1 of a tile, and where its sums go if they are a part (-1 else).
struct F8Item { int mt, nt, kb0, kb1, part; };
__device__ __forceinline__ F8Item item_at(const Fp8Dev& p, int item) {
  F8Item w;
  const int t = item - p.whole, tile = t < 0 ? item : p.whole + t / p.cuts;
  tile_at(p, tile, w.mt, w.nt);
  w.part = t < 0 ? -1 : t;
  w.kb0 = 0;
  w.kb1 = p.kblocks;
  if (t >= 0) {                      // (cut between groups of four blocks, which share a word of scales)
    const int cut = t % p.cuts, groups = (p.kblocks + 3) / 4;
    w.kb0 = groups * cut / p.cuts * 4;
    w.kb1 = cut + 1 < p.cuts ? groups * (cut + 1) / p.cuts * 4 : p.kblocks;
  }
  return w;
}
// fp32 sums of e4m3 values (format 0), both operands along K.
constexpr uint32_t idesc_e4m3(int m, int n) { return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24); }

}  // namespace

template <bool F32>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(F8_THREADS, 1)
fp8_product_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmC,
                   const __grid_constant__ CUtensorMap tmParts, Fp8Dev p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_up_1024(smem_raw);
  uint8_t* slabs = smem + F8_STAGES * F8_STAGE;
  uint64_t* full = reinterpret_cast<uint64_t*>(slabs + 2 * SLAB_BYTES);
  uint64_t* done = full + F8_STAGES;       // a stage's products are in tensor memory, and the stage is free: to the producer and to the sums
  uint64_t* tempty = done + F8_STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = warp_id(), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < F8_STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&done[s], 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(&tempty[a], 16); }     // eight summing warps in each CTA
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) tmem_alloc2(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                // the peer's barriers exist before anything signals them
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  wait_for_previous();               // (launched while what makes the operands may still run)
  const int first = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;

  if (warp < 4) {
  registers_down<F8_REGS_FEW>();
  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer (both CTAs)
    const uint32_t e = elect_one();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int item = first; ok && item < p.items; item += n_pairs) {
      const F8Item w = item_at(p, item);
      const int m0 = w.mt * 256 + static_cast<int>(rank) * BM, n0 = w.nt * 256 + static_cast<int>(rank) * BM;
      for (int kb = w.kb0; kb < w.kb1; ++kb) {
        if (!mbar_wait_warp(&done[stage], phase ^ 1, abort_flag, p.status, 1)) { ok = false; break; }
        uint8_t* sA = smem + stage * F8_STAGE;
        mbar_expect_tx(&full[stage], 2 * F8_STAGE, leader ? e : 0);
        tma2_load_3d(sA, &tmA, &full[stage], kb * F8_K, m0, 0, e);
        tma2_load_3d(sA + F8_A, &tmB, &full[stage], kb * F8_K, n0, 0, e);
        if (++stage == F8_STAGES) { stage = 0; phase ^= 1; }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (leader CTA only)
    if (leader) {
      const uint32_t e = elect_one();
      constexpr uint32_t idesc = idesc_e4m3(256, 256);
      const uint64_t a_desc0 = umma_smem_desc(smem_u32(smem), 16, 1024), b_desc0 = desc_at(a_desc0, F8_A);
      const uint32_t done0 = smem_u32(done), done1 = map_to_cta(done0, 1);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int item = first; ok && item < p.items; item += n_pairs) {
        const F8Item w = item_at(p, item);
        for (int kb = w.kb0; kb < w.kb1; ++kb) {
          if (!mbar_wait_warp(&full[stage], phase, abort_flag, p.status, 2) || !mbar_wait_warp(&tempty[acc], acc_phase ^ 1, abort_flag, p.status, 2)) { ok = false; break; }
          tc_fence_after();
          const uint64_t a_desc = desc_at(a_desc0, stage * F8_STAGE), b_desc = desc_at(b_desc0, stage * F8_STAGE);
#pragma unroll
          for (int k = 0; k < 4; ++k)                // 32 values an instruction
            umma2_f8(tmem_base + static_cast<uint32_t>(acc * 256), desc_at(a_desc, k * 32), desc_at(b_desc, k * 32), idesc, k > 0 ? 1u : 0u, e);
          umma2_commit(done0 + stage * 8, e);        // to this CTA's producer and sums
          umma2_commit(done1 + stage * 8, e);        // and to the peer's
          if (++stage == F8_STAGES) { stage = 0; phase ^= 1; }
          acc ^= 1;
          if (acc == 0) acc_phase ^= 1;
        }
      }
    }
  }
  } else {
    registers_up<F8_REGS_SUMS>();
    // ------------------------------------------------------------ sums (both CTAs, own 128 rows of the tile, one a thread; 128 columns a group)
    const int ew = warp & 3, group = (warp - 4) >> 2, row_in_tile = ew * 32 + lane;
    const uint32_t tempty_lead = map_to_cta(smem_u32(tempty), 0);
    const bool issuer = ew == 0 && lane == 0;
    uint8_t* slab = slabs + group * SLAB_BYTES;
    uint8_t* my_row = slab + row_in_tile * 128;
    const uint32_t t_group = tmem_base + (static_cast<uint32_t>(ew * 32) << 16) + static_cast<uint32_t>(group * 128);
    if (issuer) tma_prefetch_desc(&tmC);
    int acc = 0, stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int item = first; ok && item < p.items; item += n_pairs) {
      const F8Item w = item_at(p, item);
      const int m0 = w.mt * 256 + static_cast<int>(rank) * BM, n0 = w.nt * 256 + group * 128;
      const int row = m0 + row_in_tile;
      const bool mine = row < p.rows && n0 < p.cols;           // (else there is nothing to scale: zeros)
      const float* sa = p.sa + static_cast<long long>(mine ? row / p.a_block : 0) * p.sa_row;
      const float* sb = p.sb + static_cast<long long>(mine ? n0 / 128 : 0) * p.sb_row;
      float next_a = sa[w.kb0 * p.sa_col], next_b = sb[w.kb0 * p.sb_col];                    // (multiplied when they are used, a block later: they take their time)
      f32x2 c[64];
#pragma unroll
      for (int j = 0; j < 64; ++j) c[j] = pack2(0.f, 0.f);
#pragma unroll 1
      for (int kb = w.kb0; kb < w.kb1; ++kb) {
        const float by = mine ? next_a * next_b : 0.f;
        const f32x2 scale = pack2(by, by);
        const int ahead = min(kb + 1, w.kb1 - 1);
        next_a = __ldg(sa + ahead * p.sa_col);
        next_b = __ldg(sb + ahead * p.sb_col);
        ok = mbar_wait(&done[stage], phase, abort_flag, p.status, 3);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        tc_fence_after();
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          uint32_t v[16];
          tmem_ld16(t_group + static_cast<uint32_t>(acc * 256) + q * 16, v);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 8; ++j) c[q * 8 + j] = fma2(pack2(v[2 * j], v[2 * j + 1]), scale, c[q * 8 + j]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_remote(tempty_lead + acc * 8);
        acc ^= 1;
        if (++stage == F8_STAGES) { stage = 0; phase ^= 1; }
      }
      // the 128 threads of a group meet on named barriers below, so they also leave together when a wait runs out
      ok = named_barrier_and(1 + 2 * group, 128, ok);
      if (!ok) break;
      if (m0 >= p.rows) continue;                              // uniform
      const bool part = w.part >= 0;                           // (all of a part is stored, which costs less than to ask)
      if (F32 || part) {
#pragma unroll
        for (int sl = 0; sl < 4; ++sl) {                       // slabs of 32 columns
          const int col = sl * 32;
          if (!part && n0 + col >= p.cols) break;
          if (issuer) tma_store_wait_read<0>();
          named_barrier(1 + 2 * group, 128);                   // the slab is free
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            float f[4];
            unpack2(c[sl * 16 + 2 * j], f[0], f[1]);
            unpack2(c[sl * 16 + 2 * j + 1], f[2], f[3]);
            *reinterpret_cast<uint4*>(my_row + ((j ^ (row_in_tile & 7)) << 4)) = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
          }
          fence_proxy_async_smem();
          named_barrier(2 + 2 * group, 128);                   // the slab is complete
          if (issuer) {
            if (part) tma_store_3d(&tmParts, slab, group * 128 + col, w.part * 256 + static_cast<int>(rank) * BM, 0);
            else tma_store_3d(&tmC, slab, n0 + col, m0, 0);
            tma_store_commit();
          }
        }
        continue;
      }
#pragma unroll
      for (int sl = 0; sl < 2; ++sl) {                         // slabs of 64 columns
        const int col = n0 + sl * 64;
        if (col >= p.cols) break;
        if (issuer) tma_store_wait_read<0>();
        named_barrier(1 + 2 * group, 128);                     // the slab is free
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint32_t o[4];
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            float lo, hi;
            unpack2(c[sl * 32 + 4 * j + t], lo, hi);
            o[t] = pack_bf16x2(lo, hi);
          }
          *reinterpret_cast<uint4*>(my_row + ((j ^ (row_in_tile & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
        }
        fence_proxy_async_smem();
        named_barrier(2 + 2 * group, 128);                     // the slab is complete
        if (issuer) {
          tma_store_3d(&tmC, slab, col, m0, 0);
          tma_store_commit();
        }
      }
    }
    if (issuer) tma_store_wait_all();
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                  // neither CTA leaves while the other may still signal or read it
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc2(tmem_base, 512);
  }
}

// ------------------------------------------------------------------------------------------------ scales that are powers of two
namespace {

constexpr int MX_THREADS = 512;      // warps 0-3: TMA, MMA, TMEM allocation, none; 4-11: epilogue, two groups of four; 12-15: scales
constexpr int MX_REGS = 128, MX_REGS_FEW = 88, MX_REGS_EPILOGUE = 168;      // at launch, and after the epilogue has got some of the others'
static_assert(2 * MX_REGS_FEW + 2 * MX_REGS_EPILOGUE <= 4 * MX_REGS, "more registers than the block was launched with");
constexpr int MX_STAGES = 3;         // of two blocks
constexpr uint32_t MX_STAGE = 2 * F8_STAGE;
constexpr int MX_SLOTS = 4;          // of scales: four blocks each, 4 columns for the rows of a and 8 for those of b
constexpr uint32_t MX_SCALES = 256, MX_SLOT = 16;      // columns of tensor memory

__device__ __forceinline__ void umma2_mx(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t tmem_sa, uint32_t tmem_sb, uint32_t accumulate,
                                         uint32_t e) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "setp.ne.b32 e, %7, 0;\n\t"
      "@e tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(tmem_sa), "r"(tmem_sb), "r"(accumulate), "r"(e)
      : "memory");
}
// Block-scaled e4m3 operands (format 0) along K, scales of eight bits of exponent (bit 23); `id`: which byte of the words of scales (bits 4-5 for b,
// 29-30 for a).
__device__ __forceinline__ uint32_t idesc_mx(int m, int n, uint32_t id) {
  return (id << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (1u << 23) | (static_cast<uint32_t>(m >> 7) << 27) | (id << 29);
}
// One 32-bit column of each of N, for this thread's lane.
__device__ __forceinline__ void tmem_st4(uint32_t taddr, const uint32_t (&v)[4]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%4], {%0,%1,%2,%3};" ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(taddr) : "memory");
}

}  // namespace

template <bool F32>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(MX_THREADS, 1)
fp8_powers_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmC,
                  const __grid_constant__ CUtensorMap tmParts, Fp8Dev p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_up_1024(smem_raw);
  uint8_t* slabs = smem + MX_STAGES * MX_STAGE;
  uint64_t* full = reinterpret_cast<uint64_t*>(slabs + 2 * SLAB_BYTES);
  uint64_t* empty = full + MX_STAGES;
  uint64_t* sfull = empty + MX_STAGES;
  uint64_t* sempty = sfull + MX_SLOTS;
  uint64_t* tfull = sempty + MX_SLOTS;
  uint64_t* tempty = tfull + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = warp_id(), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < MX_STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int s = 0; s < MX_SLOTS; ++s) { mbar_init(&sfull[s], 8); mbar_init(&sempty[s], 1); }     // the four warps of scales in each CTA
    mbar_init(tfull, 1);
    mbar_init(tempty, 16);                                                                        // eight epilogue warps in each CTA
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 2) tmem_alloc2(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                // the peer's barriers exist before anything signals them
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  wait_for_previous();               // (launched while what makes the operands may still run)
  const int first = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;

  if (warp < 4) {
    registers_down<MX_REGS_FEW>();
    if (warp == 0) {
      // ---------------------------------------------------------- TMA producer (both CTAs)
      const uint32_t e = elect_one();
      tma_prefetch_desc(&tmA);
      tma_prefetch_desc(&tmB);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int item = first; ok && item < p.items; item += n_pairs) {
        const F8Item w = item_at(p, item);
        const int m0 = w.mt * 256 + static_cast<int>(rank) * BM, n0 = w.nt * 256 + static_cast<int>(rank) * BM;
        for (int kb = w.kb0; kb < w.kb1; kb += 2) {
          if (!mbar_wait_warp(&empty[stage], phase ^ 1, abort_flag, p.status, 1)) { ok = false; break; }
          uint8_t* sA = smem + stage * MX_STAGE;
          mbar_expect_tx(&full[stage], 2 * MX_STAGE, leader ? e : 0);
#pragma unroll
          for (int half = 0; half < 2; ++half) {     // (a block behind the last one arrives as zeros)
            tma2_load_3d(sA + half * F8_STAGE, &tmA, &full[stage], (kb + half) * F8_K, m0, 0, e);
            tma2_load_3d(sA + half * F8_STAGE + F8_A, &tmB, &full[stage], (kb + half) * F8_K, n0, 0, e);
          }
          if (++stage == MX_STAGES) { stage = 0; phase ^= 1; }
        }
      }
    } else if (warp == 1 && leader) {
      // ---------------------------------------------------------- MMA issuer
      // (bound by its own instructions, some 70 cycles a product and a few hundred for what stands around it: two blocks a stage, addresses made once)
      const uint32_t e = elect_one();
      const uint64_t a_desc0 = umma_smem_desc(smem_u32(smem), 16, 1024), b_desc0 = desc_at(a_desc0, F8_A);
      const uint32_t empty0 = smem_u32(empty), empty1 = map_to_cta(empty0, 1), sempty0 = smem_u32(sempty), sempty1 = map_to_cta(sempty0, 1);
      const uint32_t tfull0 = smem_u32(tfull), tfull1 = map_to_cta(tfull0, 1);
      int stage = 0, slot = 0;
      uint32_t phase = 0, slot_phase = 0, acc_phase = 0;
      bool ok = true;
      for (int item = first; ok && item < p.items; item += n_pairs) {
        const F8Item w = item_at(p, item);
        if (!mbar_wait_warp(tempty, acc_phase ^ 1, abort_flag, p.status, 2)) break;
        uint32_t more = 0;
        for (int kb = w.kb0; kb < w.kb1; kb += 4) {
          if (!mbar_wait_warp(&sfull[slot], slot_phase, abort_flag, p.status, 2)) { ok = false; break; }
          const uint32_t t_scales = tmem_base + MX_SCALES + static_cast<uint32_t>(slot) * MX_SLOT;
#pragma unroll
          for (int pair = 0; pair < 2; ++pair) {
            if (pair == 1 && kb + 2 >= w.kb1) break;
            if (!mbar_wait_warp(&full[stage], phase, abort_flag, p.status, 2)) { ok = false; break; }
            tc_fence_after();
            const uint64_t a_desc = desc_at(a_desc0, stage * MX_STAGE), b_desc = desc_at(b_desc0, stage * MX_STAGE);
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
              for (int k = 0; k < 4; ++k) {          // 32 values an instruction
                umma2_mx(tmem_base, desc_at(a_desc, half * F8_STAGE + k * 32), desc_at(b_desc, half * F8_STAGE + k * 32), idesc_mx(256, 256, pair * 2 + half), t_scales,
                         t_scales + 4, more, e);
                more = 1;
              }
            umma2_commit(empty0 + stage * 8, e);     // this CTA's producer
            umma2_commit(empty1 + stage * 8, e);     // the peer's
            if (++stage == MX_STAGES) { stage = 0; phase ^= 1; }
          }
          if (!ok) break;
          umma2_commit(sempty0 + slot * 8, e);
          umma2_commit(sempty1 + slot * 8, e);
          if (++slot == MX_SLOTS) { slot = 0; slot_phase ^= 1; }
        }
        if (!ok) break;
        umma2_commit(tfull0, e);
        umma2_commit(tfull1, e);
        acc_phase ^= 1;
      }
    }
  } else if (warp >= 12) {
    registers_down<MX_REGS_FEW>();
    // ------------------------------------------------------------ scales (both CTAs): a lane has rows lane, lane + 32 and so on; each warp its own copy of all of them
    const uint32_t t_lanes = tmem_base + MX_SCALES + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t sfull_lead = map_to_cta(smem_u32(sfull), 0);
    int slot = 0;
    uint32_t slot_phase = 0;
    bool ok = true;
    for (int item = first; ok && item < p.items; item += n_pairs) {
      const F8Item it = item_at(p, item);
      const int m0 = it.mt * 256 + static_cast<int>(rank) * BM, n0 = it.nt * 256;
      // (loads without conditions, of places that exist, and a group ahead: each would otherwise wait for the one before.  What a row or a
      // block that is not there is scaled by does not matter, as its values are zeros, as long as it is a number.)
      const float *sa[4], *sb[2];
      int last_row = p.rows - 1;
#pragma unroll
      for (int i = 0; i < 4; ++i) sa[i] = p.sa + static_cast<long long>(min(m0 + i * 32 + lane, last_row) / p.a_block) * p.sa_row;
#pragma unroll
      for (int i = 0; i < 2; ++i) sb[i] = p.sb + static_cast<long long>(min(n0 + i * 128, p.cols - 1) / 128) * p.sb_row;
      uint32_t next[24];
      auto load = [&](int kb) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int at = min(kb + j, p.kblocks - 1);
          const long long oa = at * p.sa_col, ob = at * p.sb_col;
#pragma unroll
          for (int i = 0; i < 4; ++i) next[i * 4 + j] = __float_as_uint(__ldg(sa[i] + oa));
#pragma unroll
          for (int i = 0; i < 2; ++i) next[16 + i * 4 + j] = __float_as_uint(__ldg(sb[i] + ob));
        }
      };
      load(it.kb0);
      for (int kb = it.kb0; ok && kb < it.kb1; kb += 4) {
        uint32_t w[6];                               // four exponents each
#pragma unroll
        for (int i = 0; i < 6; ++i)
          w[i] = (next[4 * i] >> 23 & 255u) | (next[4 * i + 1] >> 23 & 255u) << 8 | (next[4 * i + 2] >> 23 & 255u) << 16 | (next[4 * i + 3] >> 23 & 255u) << 24;
        if (kb + 4 < it.kb1) load(kb + 4);
        ok = mbar_wait_warp(&sempty[slot], slot_phase ^ 1, abort_flag, p.status, 3);
        if (!ok) break;
        tc_fence_after();
        const uint32_t t = t_lanes + static_cast<uint32_t>(slot) * MX_SLOT;
        const uint32_t a4[4] = {w[0], w[1], w[2], w[3]}, b0[4] = {w[4], w[4], w[4], w[4]}, b1[4] = {w[5], w[5], w[5], w[5]};
        tmem_st4(t, a4);
        tmem_st4(t + 4, b0);
        tmem_st4(t + 8, b1);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_remote(sfull_lead + slot * 8);
        if (++slot == MX_SLOTS) { slot = 0; slot_phase ^= 1; }
      }
    }
  } else {
    registers_up<MX_REGS_EPILOGUE>();
    // ------------------------------------------------------------ epilogue (both CTAs, own 128 rows of the tile, one a thread; 128 columns a group)
    const int ew = warp & 3, group = (warp - 4) >> 2, row_in_tile = ew * 32 + lane;
    const uint32_t tempty_lead = map_to_cta(smem_u32(tempty), 0);
    const bool issuer = ew == 0 && lane == 0;
    uint8_t* slab = slabs + group * SLAB_BYTES;
    uint8_t* my_row = slab + row_in_tile * 128;
    const uint32_t t_group = tmem_base + (static_cast<uint32_t>(ew * 32) << 16) + static_cast<uint32_t>(group * 128);
    if (issuer) tma_prefetch_desc(&tmC);
    uint32_t acc_phase = 0;
    for (int item = first; item < p.items; item += n_pairs) {
      const F8Item w = item_at(p, item);
      const int m0 = w.mt * 256 + static_cast<int>(rank) * BM, n0 = w.nt * 256 + group * 128;
      // the 128 threads of a group meet on named barriers below, so they also leave together when the wait runs out
      if (!named_barrier_and(1 + 2 * group, 128, mbar_wait(tfull, acc_phase, abort_flag, p.status, 3))) break;
      acc_phase ^= 1;
      tc_fence_after();
      uint32_t c[4][32];
#pragma unroll
      for (int q = 0; q < 4; ++q) tmem_ld32(t_group + q * 32, c[q]);
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(tempty_lead);
      if (m0 >= p.rows) continue;                              // uniform
      if (F32 || w.part >= 0) {
        const bool part = w.part >= 0;                         // (all of a part is stored, which costs less than to ask)
#pragma unroll
        for (int sl = 0; sl < 4; ++sl) {                       // slabs of 32 columns
          const int col = sl * 32;
          if (!part && n0 + col >= p.cols) break;
          if (issuer) tma_store_wait_read<0>();
          named_barrier(1 + 2 * group, 128);                   // the slab is free
#pragma unroll
          for (int j = 0; j < 8; ++j)
            *reinterpret_cast<uint4*>(my_row + ((j ^ (row_in_tile & 7)) << 4)) = make_uint4(c[sl][4 * j], c[sl][4 * j + 1], c[sl][4 * j + 2], c[sl][4 * j + 3]);
          fence_proxy_async_smem();
          named_barrier(2 + 2 * group, 128);                   // the slab is complete
          if (issuer) {
            if (part) tma_store_3d(&tmParts, slab, group * 128 + col, w.part * 256 + static_cast<int>(rank) * BM, 0);
            else tma_store_3d(&tmC, slab, n0 + col, m0, 0);
            tma_store_commit();
          }
        }
        continue;
      }
#pragma unroll
      for (int sl = 0; sl < 2; ++sl) {                         // slabs of 64 columns
        const int col = n0 + sl * 64;
        if (col >= p.cols) break;
        if (issuer) tma_store_wait_read<0>();
        named_barrier(1 + 2 * group, 128);                     // the slab is free
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint32_t o[4];
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const int at = 8 * j + 2 * t;
            o[t] = pack_bf16x2(__uint_as_float(c[2 * sl + at / 32][at % 32]), __uint_as_float(c[2 * sl + at / 32][at % 32 + 1]));
          }
          *reinterpret_cast<uint4*>(my_row + ((j ^ (row_in_tile & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
        }
        fence_proxy_async_smem();
        named_barrier(2 + 2 * group, 128);                     // the slab is complete
        if (issuer) {
          tma_store_3d(&tmC, slab, col, m0, 0);
          tma_store_commit();
        }
      }
    }
    if (issuer) tma_store_wait_all();
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                  // neither CTA leaves while the other may still signal or read it
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc2(tmem_base, 512);
  }
}

// The tiles that were cut: their parts, of 256 x 256, added up first to last.
template <typename T>
__global__ void __launch_bounds__(256) fp8_join_kernel(const float* __restrict__ parts, T* __restrict__ c, long long ld_c, Fp8Dev p) {
  constexpr int PER_TILE = 256 * 64;                           // groups of four columns
  const int at = blockIdx.x * 256 + threadIdx.x, tile = at / PER_TILE, e = at - tile * PER_TILE;
  int mt, nt;
  tile_at(p, p.whole + tile, mt, nt);
  const int r = e >> 6, col = nt * 256 + (e & 63) * 4;
  const long long row = mt * 256LL + r;
  if (row >= p.rows || col >= p.cols) return;
  const float4* src = reinterpret_cast<const float4*>(parts) + static_cast<long long>(tile) * p.cuts * PER_TILE + e;
  float4 v = src[0];
#pragma unroll 4
  for (int k = 1; k < p.cuts; ++k) {
    const float4 u = src[static_cast<long long>(k) * PER_TILE];
    v.x += u.x; v.y += u.y; v.z += u.z; v.w += u.w;
  }
  // (rows of c hold whole groups of 16 bytes)
  if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(c + row * ld_c + col) = v;
  else *reinterpret_cast<uint2*>(c + row * ld_c + col) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
}

static CUtensorMap bytes_map(const Fp8Matrix& m) {
  const uint64_t dims[3] = {static_cast<uint64_t>(m.cols), static_cast<uint64_t>(m.rows), 1};
  const uint64_t strides[2] = {static_cast<uint64_t>(m.ld), static_cast<uint64_t>(m.ld) * static_cast<uint64_t>(m.rows)};
  const uint32_t box[3] = {F8_K, BM, 1};
  return make_tmap(m.values, 3, dims, strides, box, 1, true);
}

// A launch that may begin before the kernel before it has ended (it waits for it itself).
template <class... Params, class... Args>
static cudaError_t launch_over(void (*kernel)(Params...), int blocks, int threads, size_t smem, cudaStream_t s, const Args&... args) {
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}
static void check(cudaError_t e) {
  if (e != cudaSuccess) throw std::runtime_error(std::string("himuon fp8_product: ") + cudaGetErrorString(e));
}

// How the last round of tiles is cut along the inner dimension, where less than half of the pairs would have one: into as many parts as there are pairs
// for, of 8 blocks or more.  Writing the parts and adding them up takes about as long as 20 blocks of products.  256 x 2560 x 9728 (10 tiles) 31 -> 20 us,
// 9728 x 2560 x 8192 (380 tiles on 74 pairs) 155 -> 151: large products are held back by power more than by their last round.
static void plan_cuts(Fp8Dev& p, int pairs) {
  const int total = p.tiles_m * p.tiles_n, rest = total % pairs;
  p.whole = p.items = total;
  p.cuts = 1;
  if (rest == 0 || 2 * rest > pairs) return;
  const int cuts = pairs / rest < p.kblocks / 8 ? pairs / rest : p.kblocks / 8;
  if (cuts < 2 || p.kblocks - p.kblocks / cuts < 20) return;
  p.whole = total - rest;
  p.cuts = cuts;
  p.items = p.whole + rest * cuts;
}

template <bool POWERS, bool F32>
static void launch(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc, Fp8Dev p, void* c, long long ld_c, float* parts, cudaStream_t s) {
  constexpr size_t SMEM = 1024 + F8_STAGES * F8_STAGE + 2 * SLAB_BYTES + 256;
  static_assert(MX_STAGES * MX_STAGE == F8_STAGES * F8_STAGE);
  static_assert(SMEM <= 232448, "shared memory budget of one CTA exceeded");
  static std::atomic<int> most[64] = {};
  const auto kernel = [] {
    if constexpr (POWERS) return fp8_powers_kernel<F32>;
    else return fp8_product_kernel<F32>;
  }();
  constexpr int THREADS = POWERS ? MX_THREADS : F8_THREADS;
  check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(SMEM)));
  const int pairs = pairs_at_once(kernel, THREADS, SMEM, most), most_pairs = pairs < num_sms() / 2 ? pairs : num_sms() / 2;
  plan_cuts(p, parts ? most_pairs : 1);                  // (as many parts as fp8_parts_floats() counts)
  CUtensorMap tp = tc;
  const int n = p.items - p.whole;
  if (n) {
    const uint64_t dims[3] = {256, static_cast<uint64_t>(n) * 256, 1};
    const uint64_t strides[2] = {256 * sizeof(float), dims[1] * 256 * sizeof(float)};
    const uint32_t box[3] = {32, BM, 1};
    tp = make_tmap(parts, 3, dims, strides, box, 4, true);
  }
  check(launch_over(kernel, 2 * (p.items < pairs ? p.items : pairs), THREADS, SMEM, s, ta, tb, tc, tp, p));
  if (n) {
    using T = std::conditional_t<F32, float, __nv_bfloat16>;
    fp8_join_kernel<T><<<n / p.cuts * 64, 256, 0, s>>>(parts, static_cast<T*>(c), ld_c, p);
    check(cudaGetLastError());
  }
}

long long fp8_parts_floats(const Fp8Matrix& a, const Fp8Matrix& b) {
  return a.cols > 20 * F8_K && a.rows > 0 && b.rows > 0 ? static_cast<long long>(num_sms() / 2) * 256 * 256 : 0;
}

void fp8_product(const Fp8Matrix& a, const Fp8Matrix& b, void* c, long long ld_c, int out_fp32, int powers, float* parts, cudaStream_t s) {
  const int esz = out_fp32 ? 4 : 2;
  if (a.rows <= 0 || b.rows <= 0 || a.cols <= 0 || a.cols != b.cols || b.block_rows != 128 || ld_c < b.rows || ld_c * esz % 16)
    throw std::runtime_error("himuon fp8_product: bad sizes");
  Fp8Dev p{};
  p.sa = a.scales; p.sb = b.scales;
  p.sa_row = a.scale_row; p.sa_col = a.scale_col; p.sb_row = b.scale_row; p.sb_col = b.scale_col;
  p.a_block = a.block_rows;
  p.rows = a.rows; p.cols = b.rows;
  p.tiles_m = (a.rows + 255) / 256;
  p.tiles_n = (b.rows + 255) / 256;
  p.kblocks = (a.cols + F8_K - 1) / F8_K;
  p.band = F8_BAND;
  p.status = status_word_ptr();
  if (static_cast<long long>(p.tiles_m) * p.tiles_n >= (1LL << 30)) throw std::runtime_error("himuon fp8_product: too many tiles for one launch");
  const uint64_t dims[3] = {static_cast<uint64_t>(b.rows), static_cast<uint64_t>(a.rows), 1};
  const uint64_t strides[2] = {static_cast<uint64_t>(ld_c) * esz, static_cast<uint64_t>(ld_c) * esz * dims[1]};
  const uint32_t box[3] = {static_cast<uint32_t>(128 / esz), BM, 1};
  const CUtensorMap ta = bytes_map(a), tb = bytes_map(b), tc = make_tmap(c, 3, dims, strides, box, esz, true);
  const auto run = powers ? (out_fp32 ? launch<true, true> : launch<true, false>) : (out_fp32 ? launch<false, true> : launch<false, false>);
  run(ta, tb, tc, p, c, ld_c, parts, s);
}

}  // namespace himuon
