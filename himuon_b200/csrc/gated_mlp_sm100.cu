// The gated feed-forward block  y = (act(x Wg^T) * (x Wu^T)) Wd^T  on CTA pairs: its two products with an activation in between.
//
//   UP:         g = x Wg^T and u = x Wu^T for the same 256 rows and 128 features meet in one accumulator (one CTA of the pair stages rows of
//               Wg, the other of Wu), whose epilogue writes h = act(g) * u; g and u only where a gradient will want them, 24 bits of each.
//   DOWN_GRAD:  dh = dy Wd, from whose fp32 accumulator the epilogue writes dg = dh u act'(g) and du = dh act(g), operands of the products
//               that follow, in bf16.  dh itself is never written.
//
// h, dg and du are rounded to bf16: they are the operands of the next products, and each is off by at most 2^-8 of itself, as the results are.
// Everything between two products is fp32.
//
// The main loop is the pair GEMM's (gemm2_sm100.cu has its protocol): six stages of 64 along the inner dimension (five in DOWN_GRAD), two accumulators of 256
// columns, so that one tile's epilogue runs beside the products of the next.  In DOWN_GRAD the epilogue's g and u come by TMA, a slab ahead, into the
// shared memory that dg and du leave from: with loads by the threads, which have a row each, it took longer than the products (8192 x 2560 x 9728 482 us, 377 so).
#include "activations.cuh"
#include "gated_mlp.h"
#include "gemm_epilogue.cuh"
#include "himuon.h"
#include "kernel_host.h"
#include "pair_common.cuh"
#include "sm100_common.cuh"
#include "tma_host.h"

#include <atomic>

namespace himuon {

namespace {

constexpr int GM_THREADS = 384;      // warps 0-3: TMA, MMA, TMEM allocation, none; 4-11: epilogue, two groups of four
constexpr int stages_of(int mode) { return mode == 0 ? 6 : 5; }
constexpr int slabs_of(int mode) { return mode == 0 ? 1 : 2; }      // of each epilogue group
// Registers of a thread at launch, and after the first four warps have given some to the others.
constexpr int GM_REGS = 168, GM_REGS_FEW = 104, GM_REGS_EPILOGUE = 200;
static_assert(GM_REGS_FEW + 2 * GM_REGS_EPILOGUE <= 3 * GM_REGS, "more registers than the block was launched with");
constexpr uint32_t GM_A = BM * BK * 2, GM_STAGE = 2 * GM_A;      // 128 rows of each operand, a CTA

enum { UP, DOWN_GRAD };

struct GatedDev {
  uint8_t* gu_low;                     // the lower bits of g | u; UP: null where g and u are not wanted
  int rows, inter, low, tiles_m, tiles_n, kblocks;
  int* status;
};

// A slab of 128 rows by 64 columns on its way to global memory by TMA: the 128 threads of a group, one row each.
__device__ __forceinline__ void slab_free(int group, bool issuer) {
  if (issuer) tma_store_wait_read<0>();
  named_barrier(1 + 2 * group, 128);
}
// Columns 8 j to 8 j + 7 of a row.
__device__ __forceinline__ uint4* slab_cell(uint8_t* slab, int row, int j) { return reinterpret_cast<uint4*>(slab + row * 128 + ((j ^ (row & 7)) << 4)); }
// Columns 16 q to 16 q + 15 of a thread's row.
__device__ __forceinline__ void put16(uint8_t* slab, int row, int q, const uint32_t (&o)[8]) {
#pragma unroll
  for (int j = 0; j < 2; ++j)
    *slab_cell(slab, row, 2 * q + j) = make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
}
__device__ __forceinline__ void slab_store(const CUtensorMap* tm, const uint8_t* slab, int group, int col, int row0, bool issuer) {
  fence_proxy_async_smem();
  named_barrier(2 + 2 * group, 128);                  // the slab is complete
  if (issuer) {
    tma_store_3d(tm, slab, col, row0, 0);
    tma_store_commit();
  }
}
__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
// Two kept values from a word of upper bits and the word that has their lower ones (in its first or second half).
__device__ __forceinline__ void from_kept(uint32_t upper, uint32_t low, int half, float& a, float& b) {
  a = __uint_as_float(__byte_perm(upper, low, half ? 0x1062 : 0x1040) & 0xFFFFFF00u);
  b = __uint_as_float(__byte_perm(upper, low, half ? 0x3272 : 0x3252) & 0xFFFFFF00u);
}

// 8 consecutive fp32 columns of this thread's TMEM lane.
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&v)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "r"(taddr)
               : "memory");
}
// What is kept of eight values.
__device__ __forceinline__ void put_kept(uint16_t* upper, uint8_t* low, const uint32_t (&v)[8]) {
  uint32_t o[4], l[2];
#pragma unroll
  for (int j = 0; j < 4; ++j) o[j] = __byte_perm(v[2 * j], v[2 * j + 1], 0x7632);
#pragma unroll
  for (int j = 0; j < 2; ++j) l[j] = __byte_perm(__byte_perm(v[4 * j], v[4 * j + 1], 0x0051), __byte_perm(v[4 * j + 2], v[4 * j + 3], 0x0051), 0x5410);
  *reinterpret_cast<uint4*>(upper) = make_uint4(o[0], o[1], o[2], o[3]);
  *reinterpret_cast<uint2*>(low) = make_uint2(l[0], l[1]);
}

}  // namespace

// tmA: rows of x or dy.  UP: tmB0 and tmB1 rows of Wg and Wu along the inner dimension, tmO h, tmG and tmU the halves of g | u.
// DOWN_GRAD: tmB0 Wd, its features along its rows; tmO and tmB1 the halves of what is kept of g | u, tmG and tmU those of dg | du.  (Halves have a map each: what
// a box has behind the last feature of one must not go to the first of the other.)
template <int MODE, int ACT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(GM_THREADS, 1)
gated_mlp_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB0, const __grid_constant__ CUtensorMap tmB1,
                 const __grid_constant__ CUtensorMap tmO, const __grid_constant__ CUtensorMap tmG, const __grid_constant__ CUtensorMap tmU, GatedDev p) {
  constexpr int FEATURES = MODE == UP ? 128 : 256;    // of a tile
  constexpr int GM_STAGES = stages_of(MODE), SLABS = slabs_of(MODE);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_up_1024(smem_raw);
  uint8_t* slabs = smem + GM_STAGES * GM_STAGE;
  uint64_t* full = reinterpret_cast<uint64_t*>(slabs + 2 * SLABS * SLAB_BYTES);
  uint64_t* empty = full + GM_STAGES;
  uint64_t* tfull = empty + GM_STAGES;
  uint64_t* tempty = tfull + 2;
  uint64_t* kept = tempty + 2;         // DOWN_GRAD: a slab's g and u are there, one for each epilogue group
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(kept + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = warp_id(), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  if (threadIdx.x == 0) {
    for (int g = 0; g < 2; ++g) mbar_init(&kept[g], 1);
    for (int s = 0; s < GM_STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(&tfull[a], 1); mbar_init(&tempty[a], 16); }     // eight epilogue warps in each CTA
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 2) tmem_alloc2(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                // the peer's barriers exist before anything signals them
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  const int first = blockIdx.x >> 1, n_pairs = gridDim.x >> 1, total = p.tiles_m * p.tiles_n;

  if (warp < 4) {
  registers_down<GM_REGS_FEW>();
  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer (both CTAs)
    const uint32_t e = elect_one();
    const CUtensorMap* tmB = MODE == DOWN_GRAD || rank == 0 ? &tmB0 : &tmB1;
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(tmB);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int tile = first; ok && tile < total; tile += n_pairs) {
      const int nt = tile / p.tiles_m, m0 = (tile - nt * p.tiles_m) * 2 * BM + static_cast<int>(rank) * BM;
      const int n0 = MODE == UP ? nt * 128 : nt * 256 + static_cast<int>(rank) * 128;
      for (int kb = 0; kb < p.kblocks; ++kb) {
        if (!mbar_wait_warp(&empty[stage], phase ^ 1, abort_flag, p.status, 1)) { ok = false; break; }
        uint8_t* sA = smem + stage * GM_STAGE;
        mbar_expect_tx(&full[stage], 2 * GM_STAGE, leader ? e : 0);
        tma2_load_3d(sA, &tmA, &full[stage], kb * BK, m0, 0, e);
        if (MODE == UP) {
          tma2_load_3d(sA + GM_A, tmB, &full[stage], kb * BK, n0, 0, e);
        } else {
#pragma unroll
          for (int j = 0; j < 2; ++j) tma2_load_3d(sA + GM_A + j * BK * 128, tmB, &full[stage], n0 + j * 64, kb * BK, 0, e);
        }
        if (++stage == GM_STAGES) { stage = 0; phase ^= 1; }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (leader CTA only)
    if (leader) {
      const uint32_t e = elect_one();
      constexpr uint32_t idesc = umma_idesc_bf16(2 * BM, 256, false, MODE == DOWN_GRAD);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int tile = first; ok && tile < total; tile += n_pairs) {
        if (!mbar_wait_warp(&tempty[acc], acc_phase ^ 1, abort_flag, p.status, 2)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * 256);
        for (int kb = 0; kb < p.kblocks; ++kb) {
          if (!mbar_wait_warp(&full[stage], phase, abort_flag, p.status, 2)) { ok = false; break; }
          tc_fence_after();
          const uint32_t a_base = smem_u32(smem + stage * GM_STAGE);
          const uint64_t a_desc = umma_smem_desc(a_base, 16, 1024);
          const uint64_t b_desc = umma_smem_desc(a_base + GM_A, MODE == DOWN_GRAD ? BK * 128 : 16, 1024);
#pragma unroll
          for (int k = 0; k < BK / 16; ++k)
            umma2_ss(d_tmem, desc_at(a_desc, k * 32), desc_at(b_desc, k * (MODE == DOWN_GRAD ? 2048 : 32)), idesc, (kb > 0 || k > 0) ? 1u : 0u, e);
          const uint32_t e_addr = smem_u32(&empty[stage]);
          umma2_commit(e_addr, e);                  // this CTA's producer
          umma2_commit(map_to_cta(e_addr, 1), e);   // the peer's producer
          if (++stage == GM_STAGES) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        const uint32_t f_addr = smem_u32(&tfull[acc]);
        umma2_commit(f_addr, e);
        umma2_commit(map_to_cta(f_addr, 1), e);
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
      }
    }
  }
  } else {
    registers_up<GM_REGS_EPILOGUE>();
    // ------------------------------------------------------------ epilogue (both CTAs, own 128 accumulator rows, one a thread)
    const int ew = warp & 3, group = (warp - 4) >> 2, row_in_tile = ew * 32 + lane;
    const uint32_t tempty_lead = map_to_cta(smem_u32(tempty), 0);
    const bool issuer = ew == 0 && lane == 0;
    bool ok = true;
    uint8_t* slab = slabs + group * SLABS * SLAB_BYTES;
    if (issuer) tma_prefetch_desc(&tmO);
    int acc = 0;
    uint32_t acc_phase = 0, kept_phase = 0;
    // DOWN_GRAD: the group's next slab, from columns c of a tile on (a tile may have none), and its g and u, which are on their way a slab ahead
    auto next_slab = [&](int tile, int c, int& row, int& col) {
      for (; tile < total; tile += n_pairs, c = group * 64) {
        const int nt = tile / p.tiles_m;
        row = (tile - nt * p.tiles_m) * 2 * BM + static_cast<int>(rank) * BM;
        col = nt * FEATURES + c;
        if (c < 256 && row < p.rows && col < p.inter) return true;
      }
      return false;
    };
    uint4 gl[4], ul[4];
    auto load_low = [&](int tile, int c) {
      int row, col;
      const bool there = next_slab(tile, c, row, col) && row + row_in_tile < p.rows;
      const uint8_t* low = p.gu_low + static_cast<long long>(there ? row + row_in_tile : 0) * 2 * p.low + (there ? col : 0);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const bool in = there && col + q * 16 < p.inter;
        gl[q] = in ? *reinterpret_cast<const uint4*>(low + q * 16) : make_uint4(0, 0, 0, 0);
        ul[q] = in ? *reinterpret_cast<const uint4*>(low + p.low + q * 16) : make_uint4(0, 0, 0, 0);
      }
    };
    auto load_kept = [&](int tile, int c) {
      int row, col;
      if (!next_slab(tile, c, row, col)) return;
      mbar_expect_tx(&kept[group], 2 * SLAB_BYTES);
      tma_load_3d(slab, &tmO, &kept[group], col, row, 0);
      tma_load_3d(slab + SLAB_BYTES, &tmB1, &kept[group], col, row, 0);
    };
    if constexpr (MODE == DOWN_GRAD) {
      if (issuer) load_kept(first, group * 64);
      load_low(first, group * 64);
    }
    for (int tile = first; tile < total; tile += n_pairs) {
      const int nt = tile / p.tiles_m, m0 = (tile - nt * p.tiles_m) * 2 * BM + static_cast<int>(rank) * BM;
      const int n0 = nt * FEATURES;
      // the 128 threads of a group meet on named barriers below, so they also leave together when the wait runs out
      if (!named_barrier_and(1 + 2 * group, 128, mbar_wait(&tfull[acc], acc_phase, abort_flag, p.status, 3))) break;
      tc_fence_after();
      const uint32_t t_acc = tmem_base + (static_cast<uint32_t>(ew * 32) << 16) + static_cast<uint32_t>(acc * 256);
      if (m0 < p.rows) {                            // uniform: the second CTA of a ragged last row block has nothing to store
        if constexpr (MODE == UP) {
          const int col = n0 + group * 64;
          if (col < p.inter) {
            // (values go to the slab as they come: 64 of them at once are more registers than there are)
            const uint32_t t_slab = t_acc + group * 64;
            slab_free(group, issuer);
#pragma unroll 1
            for (int q = 0; q < 4; ++q) {
              uint32_t g[16], u[16], o[8];
              tmem_ld16(t_slab + q * 16, g);
              tmem_ld16(t_slab + 128 + q * 16, u);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 8; ++j)
                o[j] = pack_bf16x2(activate<ACT>(__uint_as_float(g[2 * j])) * __uint_as_float(u[2 * j]),
                                   activate<ACT>(__uint_as_float(g[2 * j + 1])) * __uint_as_float(u[2 * j + 1]));
              put16(slab, row_in_tile, q, o);
            }
            slab_store(&tmO, slab, group, col, m0, issuer);
            if (p.gu_low) {
              uint8_t* low = p.gu_low + static_cast<long long>(m0 + row_in_tile) * 2 * p.low + col;
              const bool row_ok = m0 + row_in_tile < p.rows;
#pragma unroll 1
              for (int part = 0; part < 2; ++part) {
                slab_free(group, issuer);
#pragma unroll 1
                for (int q = 0; q < 4; ++q) {
                  uint32_t v[16], o[8], l[4];
                  tmem_ld16(t_slab + part * 128 + q * 16, v);
                  tmem_ld_wait();
#pragma unroll
                  for (int j = 0; j < 8; ++j) o[j] = __byte_perm(v[2 * j], v[2 * j + 1], 0x7632);
#pragma unroll
                  for (int j = 0; j < 4; ++j)
                    l[j] = __byte_perm(__byte_perm(v[4 * j], v[4 * j + 1], 0x0051), __byte_perm(v[4 * j + 2], v[4 * j + 3], 0x0051), 0x5410);
                  put16(slab, row_in_tile, q, o);
                  if (row_ok && col + q * 16 < p.inter) *reinterpret_cast<uint4*>(low + part * p.low + q * 16) = make_uint4(l[0], l[1], l[2], l[3]);
                }
                slab_store(part ? &tmU : &tmG, slab, group, col, m0, issuer);
              }
            }
          }
        } else {
#pragma unroll 1
          for (int c = group * 64; c < 256; c += 128) {
            const int col = n0 + c;
            if (col >= p.inter) break;                // uniform over the group
            if (!named_barrier_and(1 + 2 * group, 128, mbar_wait(&kept[group], kept_phase, abort_flag, p.status, 3))) { ok = false; break; }
            kept_phase ^= 1;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              uint4 gv[2], uv[2];
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                gv[j] = *slab_cell(slab, row_in_tile, 2 * q + j);
                uv[j] = *slab_cell(slab + SLAB_BYTES, row_in_tile, 2 * q + j);
              }
              uint32_t d[16], dg[8], du[8];
              tmem_ld16(t_acc + c + q * 16, d);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                float g0, g1, u0, u1, a0, a1, s0, s1;
                from_kept(word(gv[j / 4], j & 3), word(gl[q], j / 2), j & 1, g0, g1);
                from_kept(word(uv[j / 4], j & 3), word(ul[q], j / 2), j & 1, u0, u1);
                activate_grad<ACT>(g0, a0, s0);
                activate_grad<ACT>(g1, a1, s1);
                const float d0 = __uint_as_float(d[2 * j]), d1 = __uint_as_float(d[2 * j + 1]);
                dg[j] = pack_bf16x2(d0 * u0 * s0, d1 * u1 * s1);
                du[j] = pack_bf16x2(d0 * a0, d1 * a1);
              }
              put16(slab, row_in_tile, q, dg);
              put16(slab + SLAB_BYTES, row_in_tile, q, du);
            }
            load_low(tile, c + 128);
            fence_proxy_async_smem();
            named_barrier(2 + 2 * group, 128);        // both slabs are complete
            if (issuer) {
              tma_store_3d(&tmG, slab, col, m0, 0);
              tma_store_3d(&tmU, slab + SLAB_BYTES, col, m0, 0);
              tma_store_commit();
              tma_store_wait_read<0>();
              load_kept(tile, c + 128);
            }
          }
          if (!ok) break;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(tempty_lead + acc * 8);
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
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

// UP for up to 256 rows, whose weights are all that counts.  Tiles of 128 features would be a little more than there are pairs (76 on 74 for 9728), and the second round as
// long as the first; so a CTA by itself takes as many features as give every SM a tile (`features`, a multiple of 8), for all the rows: MT tiles of 128, which
// share the rows of Wg and Wu that it has staged.  g and u of a feature are columns of one accumulator row.  The results are few, and go straight to memory.
// 2560 x 9728 gated and back: 100 rows 45 us, 59 in tiles for pairs, 192 rows 50 and 60.
constexpr int GR_STAGES = 8, GR_SMEM = 1024 + 216 * 1024 + 256;
struct GatedRowsDev {
  void *h, *gu;
  uint8_t* gu_low;                     // null where g and u are not wanted
  int rows, inter, low, features, tiles, kblocks, stages;
  int* status;
};
template <int ACT, int MT>
__global__ void __launch_bounds__(GM_THREADS, 1)
gated_rows_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmG, const __grid_constant__ CUtensorMap tmU, GatedRowsDev p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_up_1024(smem_raw);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + 216 * 1024);
  uint64_t* empty = full + GR_STAGES;
  uint64_t *tfull = empty + GR_STAGES, *tempty = tfull + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = warp_id(), lane = threadIdx.x & 31;
  const uint32_t w_bytes = static_cast<uint32_t>(p.features) * 128, stage_bytes = MT * GM_A + 2 * w_bytes;
  if (threadIdx.x == 0) {
    for (int i = 0; i < p.stages; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    mbar_init(tfull, 1);
    mbar_init(tempty, 8);              // epilogue warps
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 2) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);

  if (warp == 0) {
    const uint32_t e = elect_one();
    tma_prefetch_desc(&tmX);
    tma_prefetch_desc(&tmG);
    tma_prefetch_desc(&tmU);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int tile = blockIdx.x; ok && tile < p.tiles; tile += gridDim.x) {
      const int n0 = tile * p.features;
      for (int kb = 0; kb < p.kblocks; ++kb) {
        if (!mbar_wait_warp(&empty[stage], phase ^ 1, abort_flag, p.status, 1)) { ok = false; break; }
        uint8_t* at = smem + stage * stage_bytes;
        mbar_expect_tx(&full[stage], stage_bytes, e);
        tma_load_3d(at + MT * GM_A, &tmG, &full[stage], kb * BK, n0, 0, e);
        tma_load_3d(at + MT * GM_A + w_bytes, &tmU, &full[stage], kb * BK, n0, 0, e);
#pragma unroll
        for (int t = 0; t < MT; ++t) tma_load_3d(at + t * GM_A, &tmX, &full[stage], kb * BK, t * BM, 0, e);
        if (++stage == p.stages) { stage = 0; phase ^= 1; }
      }
    }
  } else if (warp == 1) {
    const uint32_t e = elect_one(), idesc = umma_idesc_bf16(BM, 2 * p.features, false, false);
    int stage = 0;
    uint32_t phase = 0, acc_phase = 0;
    bool ok = true;
    for (int tile = blockIdx.x; ok && tile < p.tiles; tile += gridDim.x) {
      if (!mbar_wait_warp(tempty, acc_phase ^ 1, abort_flag, p.status, 2)) break;
      tc_fence_after();
      for (int kb = 0; kb < p.kblocks; ++kb) {
        if (!mbar_wait_warp(&full[stage], phase, abort_flag, p.status, 2)) { ok = false; break; }
        tc_fence_after();
        const uint64_t a_desc = umma_smem_desc(smem_u32(smem + stage * stage_bytes), 16, 1024), b_desc = desc_at(a_desc, MT * GM_A);
#pragma unroll
        for (int k = 0; k < BK / 16; ++k)
#pragma unroll
          for (int t = 0; t < MT; ++t)
            umma_ss(tmem_base + static_cast<uint32_t>(t * 256), desc_at(a_desc, t * GM_A + k * 32), desc_at(b_desc, k * 32), idesc, (kb > 0 || k > 0) ? 1u : 0u, e);
        umma_commit(&empty[stage], e);
        if (++stage == p.stages) { stage = 0; phase ^= 1; }
      }
      if (!ok) break;
      umma_commit(tfull, e);
      acc_phase ^= 1;
    }
  } else if (warp >= 4) {
    // one row a thread; two groups of warps have a tile of rows each, or every other eight features of the one
    const int ew = warp & 3, group = (warp - 4) >> 2, mt = MT == 2 ? group : 0, row = mt * BM + ew * 32 + lane;
    const bool row_ok = row < p.rows;
    const uint32_t t_acc = tmem_base + (static_cast<uint32_t>(ew * 32) << 16) + static_cast<uint32_t>(mt * 256);
    uint32_t acc_phase = 0;
    for (int tile = blockIdx.x; tile < p.tiles; tile += gridDim.x) {
      if (!mbar_wait_warp(tfull, acc_phase, abort_flag, p.status, 3)) break;
      acc_phase ^= 1;
      tc_fence_after();
#pragma unroll 1
      for (int c = MT == 2 ? 0 : group * 8; c < p.features; c += MT == 2 ? 8 : 16) {
        const int col = tile * p.features + c;
        if (col >= p.inter) break;                       // uniform
        uint32_t g[8], u[8];
        tmem_ld8(t_acc + c, g);
        tmem_ld8(t_acc + p.features + c, u);
        tmem_ld_wait();
        if (row_ok) {
          uint32_t o[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            o[j] = pack_bf16x2(activate<ACT>(__uint_as_float(g[2 * j])) * __uint_as_float(u[2 * j]), activate<ACT>(__uint_as_float(g[2 * j + 1])) * __uint_as_float(u[2 * j + 1]));
          *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.h) + static_cast<long long>(row) * p.inter + col) = make_uint4(o[0], o[1], o[2], o[3]);
          if (p.gu_low) {
            uint16_t* upper = static_cast<uint16_t*>(p.gu) + 2LL * row * p.inter + col;
            uint8_t* low = p.gu_low + 2LL * row * p.low + col;
            put_kept(upper, low, g);
            put_kept(upper + p.inter, low + p.low, u);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(tempty);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// Rows of `cols` bf16 values, boxes of 64 columns.
static CUtensorMap rows_map(const void* ptr, long long rows, long long cols, long long ld, int box_rows) {
  const uint64_t dims[3] = {static_cast<uint64_t>(cols), static_cast<uint64_t>(rows), 1};
  const uint64_t strides[2] = {static_cast<uint64_t>(ld) * 2, static_cast<uint64_t>(ld) * 2 * static_cast<uint64_t>(rows)};
  const uint32_t box[3] = {64, static_cast<uint32_t>(box_rows), 1};
  return make_tmap(ptr, 3, dims, strides, box, 2, true);
}

template <int MODE, int ACT>
static void launch(const CUtensorMap& a, const CUtensorMap& b0, const CUtensorMap& b1, const CUtensorMap& o, const CUtensorMap& g, const CUtensorMap& u,
                   GatedDev p, int inner, cudaStream_t s) {
  constexpr size_t SMEM = 1024 + stages_of(MODE) * GM_STAGE + 2 * slabs_of(MODE) * SLAB_BYTES + 256;
  static_assert(SMEM <= 232448, "shared memory budget of one CTA exceeded");
  static std::atomic<int> most[64] = {};
  const auto kernel = gated_mlp_kernel<MODE, ACT>;
  const cudaError_t set = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(SMEM));
  if (set != cudaSuccess) throw std::runtime_error(std::string("himuon gated_mlp: ") + cudaGetErrorString(set));
  const int pairs = pairs_at_once(kernel, GM_THREADS, SMEM, most);
  constexpr int FEATURES = MODE == UP ? 128 : 256;
  p.tiles_m = (p.rows + 2 * BM - 1) / (2 * BM);
  p.tiles_n = (p.inter + FEATURES - 1) / FEATURES;
  p.kblocks = (inner + BK - 1) / BK;
  p.status = status_word_ptr();
  const long long total = static_cast<long long>(p.tiles_m) * p.tiles_n;
  if (total >= (1LL << 30)) throw std::runtime_error("himuon gated_mlp: too many tiles for one launch");
  kernel<<<2 * static_cast<int>(total < pairs ? total : pairs), GM_THREADS, SMEM, s>>>(a, b0, b1, o, g, u, p);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) throw std::runtime_error(std::string("himuon gated_mlp launch failed: ") + cudaGetErrorString(e));
}
template <int MODE, class... Args>
static void launch_activation(int activation, const Args&... args) {
  switch (activation) {
    case kSilu: return launch<MODE, kSilu>(args...);
    case kGelu: return launch<MODE, kGelu>(args...);
    case kGeluTanh: return launch<MODE, kGeluTanh>(args...);
    case kRelu: return launch<MODE, kRelu>(args...);
  }
  throw std::runtime_error("himuon gated_mlp: unknown activation");
}

template <int ACT, int MT>
static void launch_rows(const GatedUpArgs& a, cudaStream_t s) {
  const auto kernel = gated_rows_kernel<ACT, MT>;
  GatedRowsDev p{};
  p.h = a.h; p.gu = a.gu; p.gu_low = static_cast<uint8_t*>(a.gu_low);
  p.rows = a.rows; p.inter = a.inter; p.low = gated_low(a.inter);
  const int sms = num_sms(), share = (a.inter + sms - 1) / sms;
  p.features = ((share + (share + 127) / 128 - 1) / ((share + 127) / 128) + 7) / 8 * 8;
  p.tiles = (a.inter + p.features - 1) / p.features;
  p.kblocks = (a.hidden + BK - 1) / BK;
  const int fit = 216 * 1024 / (MT * static_cast<int>(GM_A) + 2 * p.features * 128);
  p.stages = fit < GR_STAGES ? fit : GR_STAGES;
  p.status = status_word_ptr();
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, GR_SMEM);
  if (e == cudaSuccess) {
    kernel<<<p.tiles < sms ? p.tiles : sms, GM_THREADS, GR_SMEM, s>>>(rows_map(a.x, a.rows, a.hidden, a.ld_x, BM), rows_map(a.wg, a.inter, a.hidden, a.ld_wg, p.features),
                                                                     rows_map(a.wu, a.inter, a.hidden, a.ld_wu, p.features), p);
    e = cudaGetLastError();
  }
  if (e != cudaSuccess) throw std::runtime_error(std::string("himuon gated_mlp launch failed: ") + cudaGetErrorString(e));
}
template <int MT>
static void launch_rows(const GatedUpArgs& a, cudaStream_t s) {
  switch (a.activation) {
    case kSilu: return launch_rows<kSilu, MT>(a, s);
    case kGelu: return launch_rows<kGelu, MT>(a, s);
    case kGeluTanh: return launch_rows<kGeluTanh, MT>(a, s);
    case kRelu: return launch_rows<kRelu, MT>(a, s);
  }
  throw std::runtime_error("himuon gated_mlp: unknown activation");
}

void gated_up(const GatedUpArgs& a, cudaStream_t s) {
  if (a.rows <= 0 || a.inter <= 0 || a.hidden <= 0 || a.hidden % 8 || a.inter % 8) throw std::runtime_error("himuon gated_mlp: bad sizes");
  const long long ld = 2LL * a.inter;
  GatedDev p{};
  if ((a.gu == nullptr) != (a.gu_low == nullptr)) throw std::runtime_error("himuon gated_mlp: upper and lower bits go together");
  p.gu_low = static_cast<uint8_t*>(a.gu_low);
  p.rows = a.rows;
  p.inter = a.inter;
  p.low = gated_low(a.inter);
  if (a.rows <= BM) return launch_rows<1>(a, s);
  if (a.rows <= 2 * BM) return launch_rows<2>(a, s);
  const CUtensorMap o = rows_map(a.h, a.rows, a.inter, a.inter, BM);
  launch_activation<UP>(a.activation, rows_map(a.x, a.rows, a.hidden, a.ld_x, BM), rows_map(a.wg, a.inter, a.hidden, a.ld_wg, BM),
                        rows_map(a.wu, a.inter, a.hidden, a.ld_wu, BM), o, a.gu ? rows_map(a.gu, a.rows, a.inter, ld, BM) : o,
                        a.gu ? rows_map(static_cast<char*>(a.gu) + 2LL * a.inter, a.rows, a.inter, ld, BM) : o, p, a.hidden, s);
}

void gated_down_grad(const GatedDownGradArgs& a, cudaStream_t s) {
  if (a.rows <= 0 || a.inter <= 0 || a.hidden <= 0 || a.hidden % 8 || a.inter % 8) throw std::runtime_error("himuon gated_mlp: bad sizes");
  const long long ld = 2LL * a.inter;
  GatedDev p{};
  p.gu_low = static_cast<uint8_t*>(const_cast<void*>(a.gu_low));
  p.rows = a.rows;
  p.inter = a.inter;
  p.low = gated_low(a.inter);
  const CUtensorMap w = rows_map(a.wd, a.hidden, a.inter, a.ld_wd, BK), g = rows_map(a.dgu, a.rows, a.inter, ld, BM);
  launch_activation<DOWN_GRAD>(a.activation, rows_map(a.dy, a.rows, a.hidden, a.ld_dy, BM), w, rows_map(static_cast<const char*>(a.gu) + 2LL * a.inter, a.rows, a.inter, ld, BM),
                               rows_map(a.gu, a.rows, a.inter, ld, BM), g, rows_map(static_cast<char*>(a.dgu) + 2LL * a.inter, a.rows, a.inter, ld, BM), p, a.hidden, s);
}

}  // namespace himuon
