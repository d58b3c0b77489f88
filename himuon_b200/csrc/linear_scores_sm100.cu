// Log probability of given tokens and entropy straight from hidden states and the head's weight, and the gradient of the logits
// that they never were: a bf16 product on CTA pairs whose epilogue takes the fp32 accumulator's columns for what they are.
//
//   forward:   x = h W^T tile by tile; of each row of a tile only m = max x, s = sum e^(x-m), t = sum (x-m) e^(x-m) leave the kernel
//              (and the logit of the row's own token); linear_scores_join_kernel merges a row's tiles (formulas in token_scores.cu).
//   gradient:  dx_j = g [j = y] - p_j (g + h (log p_j + H)) as bf16, the operand of the products dx W and dx^T h that follow.  Either from the
//              same product again, or, where the forward pass could keep them, from its exponentials: e^(x - m of 64 columns) in 16 bits
//              (kept_pair: 10 bits at any size where the gradient gets 8), which the gradient then takes the place of.
//
// The product is the pair GEMM's (gemm2_sm100.cu has its protocol): 256 rows by 256 vocabulary entries per pair, six stages of 64 along
// the hidden size, two accumulators, so that the epilogue of one tile runs beside the products of the next.  The tiles of one
// vocabulary block are neighbours in the schedule: its rows of W come from memory once, the hidden states from the L2.
#include <stdint.h>

#include <atomic>

#include "gemm_epilogue.cuh"
#include "himuon.h"
#include "pair_common.cuh"
#include "sm100_common.cuh"
#include "tma_host.h"
#include "token_scores.cuh"

namespace himuon {

namespace {

constexpr int LS_THREADS = 384;      // warps 0-3: TMA, MMA, TMEM allocation, none; 4-11: epilogue, two groups of four
constexpr int LS_STAGES = 6;
// Vocabulary entries per tile.  Narrower ones fill the last round of tiles better, but cost more than that gives, also where one block
// of rows has every tile: 65 / 128 / 256 rows at 151936 x 1024 took 72 / 72 / 78 us with 256, 81 / 80 / 86 with 192, 109 / 108 / 111 with 128.
constexpr int LS_N = 256;
constexpr uint32_t LS_A = BM * BK * 2, LS_STAGE = 2 * LS_A;      // 128 rows of h and 128 of W, a CTA

// The tensor core cuts its fp32 sums off toward 0, 16 elements at a time, so that a logit comes out too small by about so much of itself for each element of the
// hidden size.  Measured, slope of the accumulators against 64 bits: 7.4e-10 to 9.6e-10 at hidden sizes of 64 to 8192 (normal operands, also with a part in
// common), 1.0e-9 to 1.4e-9 with heavy tails, 1.2e-9 to 3.9e-9 where all products are positive.  What all of them share is put back.
// At 2560 the entropy was off by 1.0e-6 of itself without.
constexpr float kShrink = 7.5e-10f;

enum { STATS, GRAD, STATS_KEPT };    // what the epilogue makes of the logits; STATS_KEPT: sums, and the exponentials

struct LinScoresDev {
  const long long* ids;
  float* slab_max;                   // STATS_KEPT: m of each (row, 64 columns)
  int slabs;
  float* part;                       // forward: m, s and t of each (part of the vocabulary, row), in three blocks of n_parts * rows
  float* target;                     // forward: the logit of each row's own id
  const float2* stats;               // gradient: as row_grad() takes them
  const float* entropy;
  const float* g_log_probs;
  const float* g_entropy;
  long long ignore;
  float regrow;                      // accumulator to logit (kShrink)
  int rows, vocab, tiles_m, tiles_n, kblocks;
  int* status;
};

// A row's sums over one part of the vocabulary.
__device__ __forceinline__ void put_sums(const LinScoresDev& p, const Sums& a, int part, int row) {
  const long long n = static_cast<long long>(p.tiles_n) * 2 * p.rows, i = static_cast<long long>(part) * p.rows + row;
  p.part[i] = a.m;
  p.part[n + i] = a.s;
  p.part[2 * n + i] = a.t;
}
// Two exponentials in 16 bits each.  They lie in 0..1, so that an fp32 word's sign and the first bit of its exponent are 0; the next 16
// are kept, 7 of the exponent and 9 of the mantissa, rounded.  (fp16 has a bit more from 1 to 6e-5, loses one with each factor of 2 below and has nothing
// under 3e-8: 17 nats beside a confident row's token.  A NaN may become a number: its row's sums are NaN, and so is the gradient.)
__device__ __forceinline__ uint32_t kept_pair(float a, float b) {
  return __byte_perm((__float_as_uint(a) << 2) + 0x8000u, (__float_as_uint(b) << 2) + 0x8000u, 0x7632);
}
__device__ __forceinline__ float2 from_kept(uint32_t w) {
  return make_float2(__uint_as_float((w << 14) & 0x3FFFC000u), __uint_as_float((w >> 2) & 0x3FFFC000u));
}
// The sums over 64 logits, and their exponentials relative to the largest, as kept_pair()s.
__device__ __forceinline__ Sums exponentials64(const float (&x)[64], uint32_t (&o)[32]) {
  const float m = largest<64>(x), base = m == -INFINITY ? 0.f : m;
  const f32x2 nbase = pack2(-base, -base), l2e = pack2(kLog2eS, kLog2eS);
  f32x2 s[2] = {pack2(0.f, 0.f), pack2(0.f, 0.f)}, t[2] = {s[0], s[0]};
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const f32x2 d = add2(pack2(x[2 * i], x[2 * i + 1]), nbase);
    float y0, y1, d0, d1;
    unpack2(mul2(d, l2e), y0, y1);
    unpack2(d, d0, d1);
    y0 = exp2f(y0);
    y1 = exp2f(y1);
    const f32x2 e = pack2(y0, y1);
    s[i & 1] = add2(s[i & 1], e);
    t[i & 1] = fma2(pack2(fmaxf(d0, kFar), fmaxf(d1, kFar)), e, t[i & 1]);
    o[i] = kept_pair(y0, y1);
  }
  float s0, s1, t0, t1;
  unpack2(add2(s[0], s[1]), s0, s1);
  unpack2(add2(t[0], t[1]), t0, t1);
  return Sums{m, s0 + s1, t0 + t1};
}

}  // namespace

template <int MODE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(LS_THREADS, 1)
linear_scores_kernel(const __grid_constant__ CUtensorMap tmH, const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmD,
                     LinScoresDev p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_up_1024(smem_raw);
  uint8_t* slabs = smem + LS_STAGES * LS_STAGE;
  uint64_t* full = reinterpret_cast<uint64_t*>(slabs + (MODE == STATS ? 0 : 2 * SLAB_BYTES));
  uint64_t* empty = full + LS_STAGES;
  uint64_t* tfull = empty + LS_STAGES;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = warp_id(), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < LS_STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
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

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer (both CTAs)
    const uint32_t e = elect_one();
    tma_prefetch_desc(&tmH);
    tma_prefetch_desc(&tmW);
    const uint32_t bytes = 2 * (LS_A + LS_N / 2 * BK * 2);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int tile = first; ok && tile < total; tile += n_pairs) {
      const int nt = tile / p.tiles_m, m0 = (tile - nt * p.tiles_m) * 2 * BM + static_cast<int>(rank) * BM;
      const int n0 = nt * LS_N + static_cast<int>(rank) * (LS_N / 2);
      for (int kb = 0; kb < p.kblocks; ++kb) {
        if (!mbar_wait_warp(&empty[stage], phase ^ 1, abort_flag, p.status, 1)) { ok = false; break; }
        uint8_t* sA = smem + stage * LS_STAGE;
        mbar_expect_tx(&full[stage], bytes, leader ? e : 0);
        tma2_load_3d(sA, &tmH, &full[stage], kb * BK, m0, 0, e);
        tma2_load_3d(sA + LS_A, &tmW, &full[stage], kb * BK, n0, 0, e);
        if (++stage == LS_STAGES) { stage = 0; phase ^= 1; }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (leader CTA only)
    if (leader) {
      const uint32_t e = elect_one();
      const uint32_t idesc = umma_idesc_bf16(2 * BM, LS_N, false, false);
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
          const uint32_t a_base = smem_u32(smem + stage * LS_STAGE);
          const uint64_t a_desc = umma_smem_desc(a_base, 16, 1024), b_desc = umma_smem_desc(a_base + LS_A, 16, 1024);
#pragma unroll
          for (int k = 0; k < BK / 16; ++k)
            umma2_ss(d_tmem, desc_at(a_desc, k * 32), desc_at(b_desc, k * 32), idesc, (kb > 0 || k > 0) ? 1u : 0u, e);
          const uint32_t e_addr = smem_u32(&empty[stage]);
          umma2_commit(e_addr, e);                  // this CTA's producer
          umma2_commit(map_to_cta(e_addr, 1), e);   // the peer's producer
          if (++stage == LS_STAGES) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        const uint32_t f_addr = smem_u32(&tfull[acc]);
        umma2_commit(f_addr, e);
        umma2_commit(map_to_cta(f_addr, 1), e);
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
      }
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------ epilogue (both CTAs, own 128 accumulator rows, one a thread)
    const int ew = warp & 3, group = (warp - 4) >> 2;
    const uint32_t tempty_lead = map_to_cta(smem_u32(tempty), 0);
    const bool issuer = ew == 0 && lane == 0;
    const f32x2 regrow = pack2(p.regrow, p.regrow);
    uint8_t* slab = slabs + group * SLAB_BYTES;
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int tile = first; tile < total; tile += n_pairs) {
      const int nt = tile / p.tiles_m, m0 = (tile - nt * p.tiles_m) * 2 * BM + static_cast<int>(rank) * BM;
      const int row = m0 + ew * 32 + lane, n0 = nt * LS_N;
      const bool row_ok = row < p.rows;
      RowGrad rg{};
      long long id = -1;
      if constexpr (MODE == GRAD) {
        if (row_ok) rg = row_grad(p.stats, p.entropy, p.ids, p.g_log_probs, p.g_entropy, p.ignore, p.vocab, row);
      } else {
        if (row_ok) id = p.ids[row];
      }
      // the 128 threads of a group meet on named barriers below, so they also leave together when the wait runs out
      if (!named_barrier_and(1 + 2 * group, 128, mbar_wait(&tfull[acc], acc_phase, abort_flag, p.status, 3))) break;
      tc_fence_after();
      const uint32_t t_acc = tmem_base + (static_cast<uint32_t>(ew * 32) << 16) + static_cast<uint32_t>(acc * 256);
      if (MODE == STATS || m0 < p.rows) {                     // uniform: the second CTA of a ragged last row block has nothing to store
        uint8_t* my_row = slab + (ew * 32 + lane) * 128;
        Sums a{-INFINITY, 0.f, 0.f};
#pragma unroll 1
        for (int c = group * 64; c < LS_N; c += 128) {
          const int col = n0 + c;
          if (col >= p.vocab) break;
          uint32_t o[32];
          if constexpr (MODE != GRAD) {
            float x[64];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              uint32_t v[32];
              tmem_ld32(t_acc + c + half * 32, v);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 32; j += 2) unpack2(mul2(pack2(v[j], v[j + 1]), regrow), x[half * 32 + j], x[half * 32 + j + 1]);
            }
            if (col + 64 > p.vocab) {
#pragma unroll
              for (int j = 0; j < 64; ++j) x[j] = col + j < p.vocab ? x[j] : -INFINITY;
            }
            const long long at = id - col;
            if (at >= 0 && at < 64 && id < p.vocab) {         // a row's own token: in one of its tiles
              float mine = x[0];
#pragma unroll
              for (int j = 1; j < 64; ++j) mine = at == j ? x[j] : mine;
              p.target[row] = mine;
            }
            const Sums b = exponentials64(x, o);
            a = merged(a, b);
            if (MODE == STATS_KEPT && row_ok) p.slab_max[static_cast<long long>(row) * p.slabs + col / 64] = b.m;
          } else {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint32_t v[32];
            tmem_ld32(t_acc + c + half * 32, v);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              float x0, x1;
              unpack2(mul2(pack2(v[j], v[j + 1]), regrow), x0, x1);
              o[half * 16 + j / 2] = pack_bf16x2(grad_of(rg, x0, col + half * 32 + j), grad_of(rg, x1, col + half * 32 + j + 1));
            }
          }
          }
          if constexpr (MODE == STATS) continue;
          if (issuer) tma_store_wait_read<0>();
          named_barrier(1 + 2 * group, 128);                  // the slab is free
#pragma unroll
          for (int j = 0; j < 8; ++j)
            *reinterpret_cast<uint4*>(my_row + ((j ^ (lane & 7)) << 4)) = make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
          fence_proxy_async_smem();
          named_barrier(2 + 2 * group, 128);                  // the slab is complete
          if (issuer) {
            tma_store_3d(&tmD, slab, col, m0, 0);
            tma_store_commit();
          }
        }
        if (MODE != GRAD && row_ok) put_sums(p, a, nt * 2 + group, row);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(tempty_lead + acc * 8);
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
    }
    if (MODE != STATS && issuer) tma_store_wait_all();
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                  // neither CTA leaves while the other may still signal or read it
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc2(tmem_base, 512);
  }
}

// ---------------------------------------------------------------- a few rows
// Up to 64 rows: the weight's bytes are all that counts, so the weight takes the 128 lanes of the accumulator and the rows its NB
// columns; a stage carries 16 KB of weight and 2, 4 or 8 of hidden states (the pair kernel spends half of its stages on rows that are not
// there).  A block streams one share of the vocabulary in tiles of `th` entries; a thread keeps the sums of its lane for
// up to 32 rows, and only at the end the 128 lanes meet.  8 rows over 151936 x 1024: 50 us (6.2 TB/s), pair kernel 99.
constexpr int FEW_STAGES = 9;
constexpr int few_threads(int nb) { return 64 + 128 * (nb > 32 ? nb / 32 : 1); }      // warp 0: TMA, 1: MMA, then four for each 32 rows
struct FewBars {
  uint64_t full[FEW_STAGES], empty[FEW_STAGES], tfull[2], tempty[2];
  uint32_t tmem_slot;
  int abort_flag;
};
// One lane's sums for CNT rows against the other lanes': every step halves the rows that a lane keeps.
template <int CNT, int O>
__device__ __forceinline__ void share_out(Sums* a, int lane) {
  if constexpr (O > 0) {
    constexpr int HALF = CNT > 1 ? CNT / 2 : 1;
    const bool up = (lane & O) != 0;
#pragma unroll
    for (int i = 0; i < HALF; ++i) {
      const Sums give = CNT > 1 && !up ? a[i + HALF * (CNT > 1)] : a[i], keep = CNT > 1 && up ? a[i + HALF * (CNT > 1)] : a[i];
      a[i] = merged(keep, Sums{__shfl_xor_sync(0xffffffffu, give.m, O), __shfl_xor_sync(0xffffffffu, give.s, O), __shfl_xor_sync(0xffffffffu, give.t, O)});
    }
    share_out<HALF, O / 2>(a, lane);
  }
}

template <int NB>
__global__ void __launch_bounds__(few_threads(NB), 1)
linear_scores_few_kernel(const __grid_constant__ CUtensorMap tmH, const __grid_constant__ CUtensorMap tmW, LinScoresDev p, int th) {
  constexpr uint32_t STAGE = LS_A + NB * BK * 2;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_up_1024(smem_raw);
  FewBars* bars = reinterpret_cast<FewBars*>(smem + FEW_STAGES * STAGE);
  Sums* s_warp = reinterpret_cast<Sums*>(bars + 1);      // [4][NB]
  constexpr int RB = NB < 32 ? NB : 32, GROUPS = NB / RB;      // rows of a thread, groups of four warps
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = warp_id(), lane = threadIdx.x & 31;
  // shares of whole groups of eight entries
  const long long units = (p.vocab + 7) / 8;
  const int v0 = static_cast<int>(units * blockIdx.x / gridDim.x) * 8, end = static_cast<int>(units * (blockIdx.x + 1) / gridDim.x) * 8;
  const int v1 = end < p.vocab ? end : p.vocab, tiles = (v1 - v0 + th - 1) / th;
  if (threadIdx.x == 0) {
    for (int i = 0; i < FEW_STAGES; ++i) { mbar_init(&bars->full[i], 1); mbar_init(&bars->empty[i], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&bars->tfull[i], 1); mbar_init(&bars->tempty[i], 128 * GROUPS); }
    bars->abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) tmem_alloc(&bars->tmem_slot, 128);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, bars->tmem_slot, 0);

  if (warp == 0) {
    const uint32_t e = elect_one();
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int i = 0; ok && i < tiles; ++i) {
      for (int kb = 0; kb < p.kblocks; ++kb) {
        if (!mbar_wait_warp(&bars->empty[stage], phase ^ 1, abort_flag, p.status, 1)) { ok = false; break; }
        uint8_t* sW = smem + stage * STAGE;
        mbar_expect_tx(&bars->full[stage], (th + NB) * BK * 2, e);
        tma_load_3d(sW, &tmW, &bars->full[stage], kb * BK, v0 + i * th, 0, e);
        tma_load_3d(sW + LS_A, &tmH, &bars->full[stage], kb * BK, 0, 0, e);
        if (++stage == FEW_STAGES) { stage = 0; phase ^= 1; }
      }
    }
  } else if (warp == 1) {
    const uint32_t e = elect_one();
    constexpr uint32_t idesc = umma_idesc_bf16(128, NB, false, false);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int i = 0; ok && i < tiles; ++i) {
      if (!mbar_wait_warp(&bars->tempty[i & 1], ((i >> 1) & 1) ^ 1, abort_flag, p.status, 2)) break;
      tc_fence_after();
      for (int kb = 0; kb < p.kblocks; ++kb) {
        if (!mbar_wait_warp(&bars->full[stage], phase, abort_flag, p.status, 2)) { ok = false; break; }
        tc_fence_after();
        const uint32_t base = smem_u32(smem + stage * STAGE);
        // (lanes from `th` on hold whatever an earlier tile left: rows of the product that nobody reads)
        const uint64_t w_desc = umma_smem_desc(base, 16, 1024), h_desc = umma_smem_desc(base + LS_A, 16, 1024);
#pragma unroll
        for (int k = 0; k < BK / 16; ++k)
          umma_ss(tmem + (i & 1) * NB, desc_at(w_desc, k * 32), desc_at(h_desc, k * 32), idesc, (kb > 0 || k > 0) ? 1u : 0u, e);
        umma_commit(&bars->empty[stage], e);
        if (++stage == FEW_STAGES) { stage = 0; phase ^= 1; }
      }
      if (ok) umma_commit(&bars->tfull[i & 1], e);
    }
  } else {
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const int c0 = (warp - 2) / 4 * RB;                 // the group's first row
    Sums a[RB];
#pragma unroll
    for (int n = 0; n < RB; ++n) a[n] = Sums{-INFINITY, 0.f, 0.f};
    int own[RB];                                  // the rows' own tokens, -1 where there is none
#pragma unroll
    for (int n = 0; n < RB; ++n) {
      const long long id = c0 + n < p.rows ? p.ids[c0 + n] : -1;
      own[n] = id >= 0 && id < p.vocab ? static_cast<int>(id) : -1;
    }
    for (int i = 0; i < tiles; ++i) {
      if (!mbar_wait(&bars->tfull[i & 1], (i >> 1) & 1, abort_flag, p.status, 3)) break;
      tc_fence_after();
      const int v = v0 + i * th + row;
      const bool mine = row < th && v < v1;
#pragma unroll
      for (int c = 0; c < RB; c += 16) {
        uint32_t x[16];
        tmem_ld16(tmem + (i & 1) * NB + lane_off + c0 + c, x);
        tmem_ld_wait();
        if (mine) {
#pragma unroll
          for (int n = 0; n < 16; ++n) {
            const float y = __uint_as_float(x[n]) * p.regrow;
            Sums& b = a[c + n];
            const float m = fmaxf(b.m, y), from = fmaxf(b.m - m, kFar), f = exp2f(from * kLog2eS);
            const float d = y - (m == -INFINITY ? 0.f : m), e = exp2f(d * kLog2eS);
            b.t = fmaf(fmaxf(d, kFar), e, f * fmaf(from, b.s, b.t));
            b.s = fmaf(b.s, f, e);
            b.m = m;
            if (own[c + n] == v) p.target[c0 + c + n] = y;
          }
        }
      }
      tc_fence_before();
      mbar_arrive(&bars->tempty[i & 1]);
    }
    share_out<RB, 16>(a, lane);
    if (RB == 32) s_warp[(warp & 3) * NB + c0 + lane] = a[0];
    else if ((lane & 1) == 0) s_warp[(warp & 3) * NB + (lane >> 1)] = a[0];
    named_barrier(1, 128 * GROUPS);
    const int n = (warp - 2) * 32 + lane;
    if (n < p.rows && n < NB) {
      Sums b = s_warp[n];
#pragma unroll
      for (int w = 1; w < 4; ++w) b = merged(b, s_warp[w * NB + n]);
      const long long all = static_cast<long long>(gridDim.x) * p.rows, at = static_cast<long long>(blockIdx.x) * p.rows + n;
      p.part[at] = b.m;
      p.part[all + at] = b.s;
      p.part[2 * all + at] = b.t;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 128);
  }
}

// Merges the parts of RB rows per block (RB neighbouring rows are neighbours in memory), in the same order on every run.
template <int RB>
__global__ void __launch_bounds__(256)
linear_scores_join_kernel(LinScoresDev p, int n_parts, float* log_probs, float* entropy, float2* stats) {
  constexpr int W = 256 / RB;
  __shared__ Sums s_sums[256];
  const int r = threadIdx.x % RB, w = threadIdx.x / RB;
  const long long row = static_cast<long long>(blockIdx.x) * RB + r;
  Sums a{-INFINITY, 0.f, 0.f};
  if (row < p.rows) {
    const long long n = static_cast<long long>(n_parts) * p.rows;
    for (int i = w; i < n_parts; i += 4 * W) {         // (loads of four parts at once: merging one by one waits for each)
      Sums b[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float* src = p.part + static_cast<long long>(i + u * W) * p.rows + row;
        b[u] = i + u * W < n_parts ? Sums{src[0], src[n], src[2 * n]} : Sums{-INFINITY, 0.f, 0.f};
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (i + u * W < n_parts) a = merged(a, b[u]);
    }
  }
  s_sums[threadIdx.x] = a;
  for (int o = W / 2; o > 0; o >>= 1) {
    __syncthreads();
    if (w < o) s_sums[threadIdx.x] = a = merged(a, s_sums[threadIdx.x + o * RB]);
  }
  if (w == 0 && row < p.rows) {
    const RowScore s = row_score(a);
    const long long id = p.ids[row];
    float lp = 0.f;
    if (id != p.ignore) lp = id >= 0 && id < p.vocab ? (p.target[row] - s.m) - s.log_s : nan_f();
    log_probs[row] = lp;
    entropy[row] = s.entropy;
    if (stats) stats[row] = make_float2(s.m, s.log_s);
  }
}

// Kept exponentials of a row into the gradient of its logits, in their place as a rule.  A thread has 8 columns, which share their 64's maximum.
__global__ void __launch_bounds__(256)
kept_to_gradient_kernel(LinScoresDev p, const uint4* kept, uint4* grad, int groups, int blocks_per_row) {
  const long long row = blockIdx.x / blocks_per_row;
  const int piece = static_cast<int>(blockIdx.x - row * blocks_per_row);
  const RowGrad r = row_grad(p.stats, p.entropy, p.ids, p.g_log_probs, p.g_entropy, p.ignore, p.vocab, row);
  uint4 raw[4];
  float f[4];                                         // log p = log e + f,  f = m of the 64 - m of the row - log s
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int i = (piece * 4 + u) * 256 + static_cast<int>(threadIdx.x);
    if (i < groups) {
      raw[u] = __ldcs(kept + row * groups + i);
      f[u] = (p.slab_max[row * p.slabs + (i >> 3)] - r.m) - r.log_s;
      f[u] = f[u] < kFar ? kFar : f[u];               // (-inf must not meet the 0 that it stands for; NaN stays)
    }
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int i = (piece * 4 + u) * 256 + static_cast<int>(threadIdx.x);
    if (i >= groups) break;
    const float scale = exp2f(f[u] * kLog2eS);
    const uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
    f32x2 d[4];
    const f32x2 by = pack2(-scale, -scale), c0 = pack2(r.c0, r.c0);
    if (r.h == 0.f) {                                 // uniform
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float2 e = from_kept(w[q]);
        d[q] = mul2(mul2(pack2(e.x, e.y), by), c0);
      }
    } else {
      const float h2 = r.h / kLog2eS;                 // c0 + h log p = (c0 + h f) + h / log2(e) * log2(e^x)
      const f32x2 h = pack2(h2, h2), c = pack2(fmaf(r.h, f[u], r.c0), fmaf(r.h, f[u], r.c0));
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float2 e = from_kept(w[q]);
        // (an exponential of 0 gets the log of the least normal number, and the product is 0 all the same)
        const f32x2 l = pack2(__log2f(fmaxf(e.x, 1.17549435e-38f)), __log2f(fmaxf(e.y, 1.17549435e-38f)));
        d[q] = mul2(mul2(pack2(e.x, e.y), by), fma2(h, l, c));
      }
    }
    uint32_t o[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float d0, d1;
      unpack2(d[q], d0, d1);
      if (r.y >> 3 == i) {                            // the group of the row's own token
        if ((r.y & 7) == 2 * q) d0 += r.g;
        if ((r.y & 7) == 2 * q + 1) d1 += r.g;
      }
      o[q] = pack_bf16x2(d0, d1);
    }
    __stcs(grad + row * groups + i, make_uint4(o[0], o[1], o[2], o[3]));
  }
}

// out = sum of n_parts fp32 matrices of n elements, in their order.
__global__ void __launch_bounds__(256)
sum_parts_kernel(const float4* __restrict__ parts, uint2* __restrict__ out, long long n4, int n_parts) {
  for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < n4; i += static_cast<long long>(gridDim.x) * 256) {
    float4 a = parts[i];
#pragma unroll 4
    for (int k = 1; k < n_parts; ++k) {
      const float4 b = parts[k * n4 + i];
      a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
    }
    out[i] = make_uint2(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w));
  }
}

static CUtensorMap rows_tmap(const void* ptr, int rows, int cols, long long ld, int box_rows) {
  const uint64_t dims[3] = {static_cast<uint64_t>(cols), static_cast<uint64_t>(rows), 1};
  const uint64_t strides[2] = {static_cast<uint64_t>(ld) * 2, static_cast<uint64_t>(ld) * 2 * static_cast<uint64_t>(rows)};
  const uint32_t box[3] = {64, static_cast<uint32_t>(box_rows), 1};
  return make_tmap(ptr, 3, dims, strides, box, 2, true);
}

// CTA pairs that can be resident at once on the current device.  (Callers and the autograd engine's threads may ask at the same time.)
template <int MODE>
static int pairs_at_once(size_t smem) {
  static std::atomic<int> most[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  const bool known = dev >= 0 && dev < 64;
  int n = known ? most[dev].load(std::memory_order_relaxed) : 0;
  if (n == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(num_sms());
    cfg.blockDim = dim3(LS_THREADS);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 2; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, linear_scores_kernel<MODE>, &cfg) != cudaSuccess || n <= 0) {
      cudaGetLastError();
      n = num_sms() / 2;
    }
    if (known) most[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

template <int MODE>
static void launch(const LinearScoreArgs& a, LinScoresDev& p, cudaStream_t s) {
  constexpr size_t SMEM = 1024 + LS_STAGES * LS_STAGE + 2 * SLAB_BYTES + 256;
  static_assert(SMEM <= 232448, "shared memory budget of one CTA exceeded");
  const cudaError_t set = cudaFuncSetAttribute(linear_scores_kernel<MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(SMEM));
  if (set != cudaSuccess) throw std::runtime_error(std::string("himuon linear_scores: ") + cudaGetErrorString(set));
  const int pairs = pairs_at_once<MODE>(SMEM);
  p.tiles_m = (p.rows + 2 * BM - 1) / (2 * BM);
  p.tiles_n = (p.vocab + LS_N - 1) / LS_N;
  p.kblocks = (a.hidden + BK - 1) / BK;
  const long long total = static_cast<long long>(p.tiles_m) * p.tiles_n;
  if (total >= (1LL << 30)) throw std::runtime_error("himuon linear_scores: too many tiles for one launch");
  const CUtensorMap th = rows_tmap(a.h, a.rows, a.hidden, a.ld_h, BM), tw = rows_tmap(a.w, a.vocab, a.hidden, a.ld_w, LS_N / 2),
                    td = MODE == STATS ? th : rows_tmap(a.grad, a.rows, static_cast<int>(a.ld_grad), a.ld_grad, BM);
  const int grid = 2 * static_cast<int>(total < pairs ? total : pairs);
  linear_scores_kernel<MODE><<<grid, LS_THREADS, SMEM, s>>>(th, tw, td, p);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) throw std::runtime_error(std::string("himuon linear_scores launch failed: ") + cudaGetErrorString(e));
}

// Returns the number of parts.
template <int NB>
static int launch_few(const LinearScoreArgs& a, LinScoresDev& p, cudaStream_t s) {
  constexpr size_t SMEM = 1024 + FEW_STAGES * (LS_A + NB * BK * 2) + sizeof(FewBars) + 4 * NB * sizeof(Sums);
  static_assert(SMEM <= 232448, "shared memory budget of one CTA exceeded");
  const cudaError_t set = cudaFuncSetAttribute(linear_scores_few_kernel<NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(SMEM));
  if (set != cudaSuccess) throw std::runtime_error(std::string("himuon linear_scores: ") + cudaGetErrorString(set));
  p.kblocks = (a.hidden + BK - 1) / BK;
  const int blocks = 2 * ((a.vocab + 127) / 128), grid = blocks < num_sms() ? blocks : num_sms();    // (scratch holds so many parts)
  const int share = ((a.vocab + 7) / 8 + grid - 1) / grid * 8, tiles = (share + 127) / 128, th = ((share + tiles - 1) / tiles + 7) / 8 * 8;
  const CUtensorMap thid = rows_tmap(a.h, a.rows, a.hidden, a.ld_h, NB), tw = rows_tmap(a.w, a.vocab, a.hidden, a.ld_w, th);
  linear_scores_few_kernel<NB><<<grid, few_threads(NB), SMEM, s>>>(thid, tw, p, th);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) throw std::runtime_error(std::string("himuon linear_scores launch failed: ") + cudaGetErrorString(e));
  return grid;
}

static LinScoresDev make_dev(const LinearScoreArgs& a) {
  if (a.rows <= 0 || a.vocab <= 0 || a.hidden <= 0 || a.hidden % 8) throw std::runtime_error("himuon linear_scores: bad sizes");
  LinScoresDev p{};
  p.ids = a.ids; p.ignore = a.ignore;
  p.rows = a.rows; p.vocab = a.vocab;
  p.regrow = 1.f + kShrink * static_cast<float>(a.hidden);
  p.part = a.scratch + a.rows; p.target = a.scratch;
  p.stats = reinterpret_cast<const float2*>(a.stats);
  p.entropy = a.entropy;
  p.g_log_probs = a.g_log_probs; p.g_entropy = a.g_entropy;
  p.status = status_word_ptr();
  return p;
}

// Room for the parts of the forward kernel that takes so many rows, one for each 64 entries (launch_few) or 128, and the rows' own logits.
long long linear_scores_scratch(long long rows, int vocab) {
  const int per = rows <= kFewRows ? 128 : LS_N;
  return rows * (1 + 3LL * 2 * ((vocab + per - 1) / per));
}

void linear_scores_fwd(const LinearScoreArgs& a, cudaStream_t s) {
  LinScoresDev p = make_dev(a);
  int n_parts;
  if (a.grad != nullptr) {
    p.slab_max = a.slab_max;
    p.slabs = (a.vocab + 63) / 64;
    launch<STATS_KEPT>(a, p, s);
    n_parts = 2 * p.tiles_n;
  } else if (a.rows <= kFewRows) {
    n_parts = a.rows <= 16 ? launch_few<16>(a, p, s) : a.rows <= 32 ? launch_few<32>(a, p, s) : launch_few<64>(a, p, s);
  } else {
    launch<STATS>(a, p, s);
    n_parts = 2 * p.tiles_n;
  }
  float2* stats = reinterpret_cast<float2*>(a.stats);
  if (a.rows < 512) linear_scores_join_kernel<1><<<a.rows, 256, 0, s>>>(p, n_parts, a.log_probs, a.entropy, stats);
  else linear_scores_join_kernel<8><<<(a.rows + 7) / 8, 256, 0, s>>>(p, n_parts, a.log_probs, a.entropy, stats);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) throw std::runtime_error(std::string("himuon linear_scores join launch failed: ") + cudaGetErrorString(e));
}

void sum_parts(const float* parts, void* out, long long n, int n_parts, cudaStream_t s) {
  if (n <= 0 || n_parts <= 0) return;
  if (n % 4) throw std::runtime_error("himuon sum_parts: a multiple of 4 elements expected");
  const long long blocks = (n / 4 + 255) / 256, most = static_cast<long long>(num_sms()) * 8;
  sum_parts_kernel<<<static_cast<int>(blocks < most ? blocks : most), 256, 0, s>>>(reinterpret_cast<const float4*>(parts), reinterpret_cast<uint2*>(out), n / 4, n_parts);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) throw std::runtime_error(std::string("himuon sum_parts launch failed: ") + cudaGetErrorString(e));
}

void linear_scores_dlogits(const LinearScoreArgs& a, cudaStream_t s) {
  LinScoresDev p = make_dev(a);
  if (a.slab_max != nullptr) {
    p.slab_max = a.slab_max;
    p.slabs = (a.vocab + 63) / 64;
    const int groups = static_cast<int>(a.ld_grad / 8), per_row = (groups + 1023) / 1024;
    if (static_cast<long long>(a.rows) * per_row >= (1LL << 31)) throw std::runtime_error("himuon linear_scores: gradient too large for one launch");
    kept_to_gradient_kernel<<<a.rows * per_row, 256, 0, s>>>(p, reinterpret_cast<const uint4*>(a.kept ? a.kept : a.grad), reinterpret_cast<uint4*>(a.grad), groups, per_row);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) throw std::runtime_error(std::string("himuon linear_scores gradient launch failed: ") + cudaGetErrorString(e));
    return;
  }
  launch<GRAD>(a, p, s);
}

}  // namespace himuon
