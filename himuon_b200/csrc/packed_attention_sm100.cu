// Causal grouped-query attention over documents of different lengths packed into one row of tokens, forward and backward.
//
//   o_i = sum_j p_ij v_j,  p_ij = softmax_j(scale q_i k_j)  over j <= i of i's own document;
//   with delta_i = sum(o_i dO_i) and dS_ij = p_ij (dO_i v_j - delta_i):   dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO.
//
// A document is cut into tiles of 128 tokens from its first token on.  The host lists the tiles of a batch once, heaviest first
// (PackedTile), every layer of a model uses the list, and a block looks its tile up: no block is launched for nothing, and the long
// ones start first.  The rows' statistics (log-sum-exp and delta) are kept by tile, 128 for each, so that
// the backward pass can fetch them in aligned bulk copies wherever a document starts.
// A TMA box is 64 or 128 tokens high whatever a document's length, so the last tile of a document brings rows of the next one
// along.  As rows of a product's result they are simply not stored; as scores they are masked like the future; but where they are
// summed over (V in P V, K in dS K, Q and dO in the dK / dV products) a probability of 0 does not make them harmless (0 times NaN), so
// the issuing warp clears them in shared memory before the product.
#include "attention_common.cuh"

#include <string>

namespace himuon {

namespace {

constexpr int BKV = 64;                              // KV positions per block of the forward pass
constexpr uint32_t KV_HALF = BKV * 128;              // one 64-column half of a K or V block: 8 KB

struct PackedDev {
  const PackedTile* tiles;
  void* o; float* lse; float* delta;
  const void* o_in;
  void* dq; void* dk; void* dv;
  int Hq, Hkv, hd;
  long long stat_rows;                               // rows of statistics per head: 128 for each tile
  long long ld_o, ld_dq, ld_dk, ld_dv;
  float scale_log2, scale;
  int* status;
};

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

// ================================================================================================ forward
struct Fwd64TBars {
  uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_ready[2], o_done[2], acc_done;
  uint32_t tmem_slot;
  int abort_flag;
};

template <int NH>
__global__ void __launch_bounds__(192, 2)
packed_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                     const __grid_constant__ CUtensorMap tmV, PackedDev p) {
  constexpr uint32_t TILE_BYTES = NH * HALF_BYTES, KV_TILE = NH * KV_HALF;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_up_1024(smem_raw);
  uint8_t* sQ = smem;                          // 32 KB
  uint8_t* sK = smem + TILE_BYTES;             // 2 stages x 16 KB
  uint8_t* sV = sK + 2 * KV_TILE;              // 2 stages x 16 KB
  Fwd64TBars* bars = reinterpret_cast<Fwd64TBars*>(sV + 2 * KV_TILE);
  volatile int* abort_flag = &bars->abort_flag;

  const int warp = warp_id(), lane = threadIdx.x & 31;
  const int order = blockIdx.x / p.Hq, h = blockIdx.x - order * p.Hq;
  const PackedTile tile = p.tiles[order];
  const int qb = tile.index, len = tile.len, first = tile.first;
  const int hk = h / (p.Hq / p.Hkv);
  int nkv = (qb + 1) * (AT / BKV);             // KV blocks up to and including the diagonal
  const int nkv_all = (len + BKV - 1) / BKV;
  if (nkv > nkv_all) nkv = nkv_all;

  auto load_k = [&](int j, uint32_t e) {
    const int st = j & 1;
    mbar_expect_tx(&bars->k_full[st], KV_TILE, e);
    load_head_tile<NH>(sK + st * KV_TILE, KV_HALF, &tmK, &bars->k_full[st], hk, first + j * BKV, 0, e);
  };
  auto load_v = [&](int j, uint32_t e) {
    const int st = j & 1;
    mbar_expect_tx(&bars->v_full[st], KV_TILE, e);
    load_head_tile<NH>(sV + st * KV_TILE, KV_HALF, &tmV, &bars->v_full[st], hk, first + j * BKV, 0, e);
  };
  if (warp == 0) {                             // the first loads are on their way while the block sets itself up
    if (lane == 0) {
      mbar_init(&bars->q_full, 1);
      for (int i = 0; i < 2; ++i) {
        mbar_init(&bars->k_full[i], 1); mbar_init(&bars->k_empty[i], 1);
        mbar_init(&bars->v_full[i], 1); mbar_init(&bars->v_empty[i], 1);
        mbar_init(&bars->s_full[i], 1); mbar_init(&bars->p_ready[i], 128);
      }
      for (int i = 0; i < 2; ++i) mbar_init(&bars->o_done[i], 1);
      mbar_init(&bars->acc_done, 1);
      bars->abort_flag = 0;
      mbar_fence_init();
    }
    __syncwarp();
    const uint32_t e = elect_one();
    mbar_expect_tx(&bars->q_full, TILE_BYTES, e);
    load_head_tile<NH>(sQ, HALF_BYTES, &tmQ, &bars->q_full, h, first + qb * AT, 0, e);
    for (int j = 0; j < 2 && j < nkv; ++j) { load_k(j, e); load_v(j, e); }
  }
  if (warp == 1) tmem_alloc(&bars->tmem_slot, 256);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, bars->tmem_slot, 0);
  const uint32_t tS0 = tmem, tO = tmem + 128;   // S / P buffers at columns 0 and 64, O at 128

  if (warp == 0) {
    const uint32_t e = elect_one();
    for (int j = 2; j < nkv; ++j) {
      const uint32_t par = ((j >> 1) & 1) ^ 1;
      if (!mbar_wait_warp(&bars->k_empty[j & 1], par, abort_flag, p.status, 4)) break;
      load_k(j, e);
      if (!mbar_wait_warp(&bars->v_empty[j & 1], par, abort_flag, p.status, 4)) break;
      load_v(j, e);
    }
  } else if (warp == 1) {
    {
      const uint32_t e = elect_one();
      constexpr uint32_t idesc_s = umma_idesc_bf16(128, BKV, false, false);
      constexpr uint32_t idesc_pv = umma_idesc_bf16(128, 64 * NH, false, true);
      const uint64_t q_desc = kmajor_desc(sQ), k_desc = kmajor_desc(sK), v_mn = mnmajor_desc(sV, KV_HALF);
      bool ok = mbar_wait_warp(&bars->q_full, 0, abort_flag, p.status, 4);
      auto issue_s = [&](int j) -> bool {
        const int st = j & 1;
        if (!mbar_wait_warp(&bars->k_full[st], (j >> 1) & 1, abort_flag, p.status, 4)) return false;
        tc_fence_after();
        // buffer st held S(j-2) / P(j-2): the softmax threads are done with it (p_ready(j-2) was waited for) and the
        // P(j-2)·V MMAs were issued earlier, which the tensor core executes in order before these
#pragma unroll
        for (int ks = 0; ks < 4 * NH; ++ks)
          umma_ss(tS0 + st * BKV, desc_at(q_desc, kmajor_off(HALF_BYTES, ks)), desc_at(k_desc, st * KV_TILE + kmajor_off(KV_HALF, ks)), idesc_s, ks > 0 ? 1u : 0u, e);
        umma_commit(&bars->k_empty[st], e);
        umma_commit(&bars->s_full[st], e);
        return true;
      };
      if (ok) ok = issue_s(0);
      for (int j = 0; ok && j < nkv; ++j) {
        if (j + 1 < nkv) { ok = issue_s(j + 1); if (!ok) break; }
        const int st = j & 1;
        if (!mbar_wait_warp(&bars->p_ready[st], (j >> 1) & 1, abort_flag, p.status, 4)) break;
        if (!mbar_wait_warp(&bars->v_full[st], (j >> 1) & 1, abort_flag, p.status, 4)) break;
        if ((j + 1) * BKV > len) clear_rows<NH>(sV + st * KV_TILE, KV_HALF, len - j * BKV, BKV, lane);
        tc_fence_after();
#pragma unroll
        for (int ks = 0; ks < BKV / 16; ++ks)
          umma_ts(tO, tS0 + st * BKV + ks * 8, desc_at(v_mn, st * KV_TILE + mnmajor_off(ks)), idesc_pv, (j > 0 || ks > 0) ? 1u : 0u, e);
        umma_commit(&bars->v_empty[st], e);
        umma_commit(&bars->o_done[st], e);
      }
      if (ok) umma_commit(&bars->acc_done, e);
    }
  } else {
    // ------------------------------------------------------------ softmax / epilogue: one thread per query row
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const int q_idx = qb * AT + row;
    float m_used = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = 0; j < nkv; ++j) {
      const int st = j & 1;
      if (!mbar_wait(&bars->s_full[st], (j >> 1) & 1, abort_flag, p.status, 4)) { ok = false; break; }
      tc_fence_after();
      const uint32_t tS = tS0 + st * BKV + lane_off;
      const int kv0 = j * BKV;
      const bool diag = (kv0 + BKV - 1 > qb * AT);       // the block reaches past the first row of this query tile
      uint32_t v0[32], v1[32];
      tmem_ld32(tS, v0);
      tmem_ld32(tS + 32, v1);
      tmem_ld_wait();
      float mx = -INFINITY;
#pragma unroll
      for (int t = 0; t < 32; ++t) {
        float s0 = __uint_as_float(v0[t]) * p.scale_log2, s1 = __uint_as_float(v1[t]) * p.scale_log2;
        if (diag && (kv0 + t > q_idx)) s0 = -INFINITY;
        if (diag && (kv0 + 32 + t > q_idx)) s1 = -INFINITY;
        v0[t] = __float_as_uint(s0);
        v1[t] = __float_as_uint(s1);
        mx = fmaxf(mx, fmaxf(s0, s1));
      }
      const float m_new = fmaxf(m_used, mx);
      const bool need = (j > 0) && (m_new - m_used > 8.f);
      const bool warp_need = __any_sync(0xffffffffu, need);
      if (j == 0) {
        m_used = m_new;
      } else if (warp_need) {
        // O (and l) move to the new maximum: the previous P·V must have landed in O first
        const float alpha = exp2f(m_used - m_new);
        m_used = m_new;
        if (!mbar_wait(&bars->o_done[st ^ 1], ((j - 1) >> 1) & 1, abort_flag, p.status, 4)) { ok = false; break; }
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < 2 * NH; ++c) {
          uint32_t v[32];
          tmem_ld32(tO + lane_off + c * 32, v);
          tmem_ld_wait();
#pragma unroll
          for (int t = 0; t < 32; ++t) v[t] = __float_as_uint(__uint_as_float(v[t]) * alpha);
          tmem_st32(tO + lane_off + c * 32, v);
        }
        l *= alpha;
      }
      uint32_t pk[32];
      float rs = 0.f;
#pragma unroll
      for (int t = 0; t < 32; t += 2) {
        // masked entries are -inf: exp2 gives exactly 0
        pk[t >> 1] = pack_bf16x2(exp2f(__uint_as_float(v0[t]) - m_used), exp2f(__uint_as_float(v0[t + 1]) - m_used));
        pk[16 + (t >> 1)] = pack_bf16x2(exp2f(__uint_as_float(v1[t]) - m_used), exp2f(__uint_as_float(v1[t + 1]) - m_used));
        rs += bf16_lo(pk[t >> 1]) + bf16_hi(pk[t >> 1]) + bf16_lo(pk[16 + (t >> 1)]) + bf16_hi(pk[16 + (t >> 1)]);
      }
      l += rs;
      tmem_st32(tS, pk);                     // P over the first 32 columns of the S buffer just read
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&bars->p_ready[st]);
    }
    if (ok && mbar_wait(&bars->acc_done, 0, abort_flag, p.status, 4)) {
      tc_fence_after();
      const float inv = 1.f / l;
      const int row0 = qb * AT + (warp & 3) * 32;
      __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(p.o) + static_cast<long long>(first + row0) * p.ld_o + h * p.hd;
      uint8_t* stage = smem + (warp & 3) * (NH * 4096);    // over Q: every product has been computed
      // Half a tile of rows or less: a thread stores its own, because turning them around takes longer than it saves (128 x 64
      // tokens, 16 heads of 128: 34.4 us, 39.0 staged; 8 x 96 already 6.5 against 6.4).  Heads of 64 gain less than the branch
      // costs their longer sequences (64 x 64 tokens 15.7 -> 15.1, but 16 x 128 6.6 -> 6.9).
      const bool few = NH == 2 && len - qb * AT <= AT / 2;
#pragma unroll 1
      for (int c = 0; c < 2 * NH; ++c) {
        uint32_t v[32];
        tmem_ld32(tO + lane_off + c * 32, v);
        tmem_ld_wait();
        if (few) {
          if (q_idx < len) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              if (c * 32 + q * 8 < p.hd) *reinterpret_cast<uint4*>(out + lane * p.ld_o + c * 32 + q * 8) = head8(v + 8 * q, inv);
          }
        } else {
          stage_head32<8 * NH>(stage, lane, c, v, inv);
        }
      }
      if (!few) store_staged<8 * NH>(out, p.ld_o, stage, lane, len - row0, p.hd);
      p.lse[h * p.stat_rows + tile.slot * AT + row] = q_idx < len ? m_used + log2f(l) : INFINITY;   // base-2 log-sum-exp of the scaled scores
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 256);
  }
}

// ================================================================================================ backward
constexpr int BQ = 64;                               // positions per streamed sub-block
constexpr uint32_t Q_HALF = BQ * 128;                // one 64-column half of a sub-block: 8 KB
constexpr int NST = 4;                               // streamed stages
constexpr uint32_t STAT_BYTES = 2 * BQ * 4;          // lse[64] then delta[64]
constexpr int BWD_THREADS = 576;                     // warp 0: TMA, warp 1: MMA issue, warps 2-17: four softmax groups
// A packed bf16 tile lies over the fp32 columns that its writers have read themselves: columns 0-15 and 32-47 of its buffer.
__device__ __forceinline__ uint32_t packed_col(int ks) { return static_cast<uint32_t>((ks >> 1) * 32 + (ks & 1) * 8); }

struct DkvBars {
  uint64_t kv_full, qd_full[NST], qd_empty[NST], s_full[2], p_ready[2], acc_done;
  uint32_t tmem_slot;
  int abort_flag;
};

__device__ __forceinline__ void bulk_load_1d(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

template <int NH>
__global__ void __launch_bounds__(BWD_THREADS, 1)
packed_dkv_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                       const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmDO, PackedDev p) {
  constexpr uint32_t TILE_BYTES = NH * HALF_BYTES, Q_TILE = NH * Q_HALF;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_up_1024(smem_raw);
  uint8_t* sK = smem;
  uint8_t* sV = smem + TILE_BYTES;
  uint8_t* sQ = smem + 2 * TILE_BYTES;                 // NST x 16 KB
  uint8_t* sDO = sQ + NST * Q_TILE;                    // NST x 16 KB
  float* sStat = reinterpret_cast<float*>(sDO + NST * Q_TILE);   // NST x (lse[64], delta[64])
  DkvBars* bars = reinterpret_cast<DkvBars*>(reinterpret_cast<uint8_t*>(sStat) + NST * STAT_BYTES);
  volatile int* abort_flag = &bars->abort_flag;

  const int warp = warp_id(), lane = threadIdx.x & 31;
  const int order = blockIdx.x / p.Hkv, hk = blockIdx.x - order * p.Hkv;
  const PackedTile tile = p.tiles[order];
  const int kb = tile.index, len = tile.len, first = tile.first;
  const int G = p.Hq / p.Hkv, h_first = hk * G;
  const int nsub = (len - kb * AT + BQ - 1) / BQ;      // query sub-blocks from the diagonal to the end
  const int iters = G * nsub;

  auto load_stage = [&](int it, uint32_t e) {
    const int g = it / nsub;
    const int h = h_first + g;
    const int q0 = kb * AT + (it - g * nsub) * BQ;
    const int st = it % NST;
    mbar_expect_tx(&bars->qd_full[st], 2 * Q_TILE + STAT_BYTES, e);
    load_head_tile<NH>(sQ + st * Q_TILE, Q_HALF, &tmQ, &bars->qd_full[st], h, first + q0, 0, e);
    load_head_tile<NH>(sDO + st * Q_TILE, Q_HALF, &tmDO, &bars->qd_full[st], h, first + q0, 0, e);
    const long long stat_idx = h * p.stat_rows + (tile.slot - kb) * AT + q0;
    if (e) bulk_load_1d(sStat + st * 2 * BQ, p.lse + stat_idx, BQ * 4, &bars->qd_full[st]);
    if (e) bulk_load_1d(sStat + st * 2 * BQ + BQ, p.delta + stat_idx, BQ * 4, &bars->qd_full[st]);
  };
  if (warp == 0) {                     // the first loads are on their way while the block sets itself up
    if (lane == 0) {
      mbar_init(&bars->kv_full, 1);
      for (int i = 0; i < NST; ++i) { mbar_init(&bars->qd_full[i], 1); mbar_init(&bars->qd_empty[i], 1); }
      for (int i = 0; i < 2; ++i) { mbar_init(&bars->s_full[i], 1); mbar_init(&bars->p_ready[i], 256); }
      mbar_init(&bars->acc_done, 1);
      bars->abort_flag = 0;
      mbar_fence_init();
    }
    __syncwarp();
    const uint32_t e = elect_one();
    mbar_expect_tx(&bars->kv_full, 2 * TILE_BYTES, e);
    load_head_tile<NH>(sK, HALF_BYTES, &tmK, &bars->kv_full, hk, first + kb * AT, 0, e);
    load_head_tile<NH>(sV, HALF_BYTES, &tmV, &bars->kv_full, hk, first + kb * AT, 0, e);
    for (int it = 0; it < NST && it < iters; ++it) load_stage(it, e);
  }
  if (warp == 1) tmem_alloc(&bars->tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, bars->tmem_slot, 0);
  const uint32_t tS = tmem, tDP = tmem + 128, tDV = tmem + 256, tDK = tmem + 384;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    const uint32_t e = elect_one();
    for (int it = NST; it < iters; ++it) {
      if (!mbar_wait_warp(&bars->qd_empty[it % NST], ((it / NST) & 1) ^ 1, abort_flag, p.status, 4)) break;
      load_stage(it, e);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issue
    {
      const uint32_t e = elect_one();
      constexpr uint32_t idesc_s = umma_idesc_bf16(128, BQ, false, false);
      constexpr uint32_t idesc_acc = umma_idesc_bf16(128, 64 * NH, false, true);
      const uint64_t k_desc = kmajor_desc(sK), v_desc = kmajor_desc(sV), q_desc = kmajor_desc(sQ), do_desc = kmajor_desc(sDO);
      const uint64_t q_mn = mnmajor_desc(sQ, Q_HALF), do_mn = mnmajor_desc(sDO, Q_HALF);
      bool ok = mbar_wait_warp(&bars->kv_full, 0, abort_flag, p.status, 4);
      auto issue_sp = [&](int it) -> bool {
        const int st = it % NST, buf = it & 1;
        if (!mbar_wait_warp(&bars->qd_full[st], (it / NST) & 1, abort_flag, p.status, 4)) return false;
        const int q0 = kb * AT + (it % nsub) * BQ;
        if (q0 + BQ > len) {
          clear_rows<NH>(sQ + st * Q_TILE, Q_HALF, len - q0, BQ, lane);
          clear_rows<NH>(sDO + st * Q_TILE, Q_HALF, len - q0, BQ, lane);
        }
        tc_fence_after();
        // The buffer's previous contents (P^T, dS^T of sub-block it-2) were consumed by MMAs issued earlier, which
        // the tensor core executes in order before these.
#pragma unroll
        for (int ks = 0; ks < 4 * NH; ++ks)
          umma_ss(tS + buf * BQ, desc_at(k_desc, kmajor_off(HALF_BYTES, ks)), desc_at(q_desc, st * Q_TILE + kmajor_off(Q_HALF, ks)), idesc_s, ks > 0 ? 1u : 0u, e);
#pragma unroll
        for (int ks = 0; ks < 4 * NH; ++ks)
          umma_ss(tDP + buf * BQ, desc_at(v_desc, kmajor_off(HALF_BYTES, ks)), desc_at(do_desc, st * Q_TILE + kmajor_off(Q_HALF, ks)), idesc_s, ks > 0 ? 1u : 0u, e);
        umma_commit(&bars->s_full[buf], e);
        return true;
      };
      if (ok) ok = issue_sp(0);
      for (int it = 0; ok && it < iters; ++it) {
        if (it + 1 < iters) { ok = issue_sp(it + 1); if (!ok) break; }
        const int st = it % NST, buf = it & 1;
        if (!mbar_wait_warp(&bars->p_ready[buf], (it >> 1) & 1, abort_flag, p.status, 4)) break;
        tc_fence_after();
#pragma unroll
        for (int ks = 0; ks < BQ / 16; ++ks)
          umma_ts(tDV, tS + buf * BQ + packed_col(ks), desc_at(do_mn, st * Q_TILE + mnmajor_off(ks)), idesc_acc, (it > 0 || ks > 0) ? 1u : 0u, e);
#pragma unroll
        for (int ks = 0; ks < BQ / 16; ++ks)
          umma_ts(tDK, tDP + buf * BQ + packed_col(ks), desc_at(q_mn, st * Q_TILE + mnmajor_off(ks)), idesc_acc, (it > 0 || ks > 0) ? 1u : 0u, e);
        umma_commit(&bars->qd_empty[st], e);
      }
      if (ok) umma_commit(&bars->acc_done, e);
    }
  } else {
    // ------------------------------------------------------------ softmax / epilogue: one thread per key row
    const int wg = (warp - 2) >> 2, buf = wg & 1, part = wg >> 1;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const int kv_idx = kb * AT + row;
    const f32x2 nscale = pack2(-p.scale_log2, -p.scale_log2), minus = pack2(-1.f, -1.f);
    bool ok = true;
    for (int it = buf; it < iters; it += 2) {
      const int g = it / nsub;
      const int q0 = kb * AT + (it - g * nsub) * BQ;
      const int st = it % NST;
      if (!mbar_wait(&bars->qd_full[st], (it / NST) & 1, abort_flag, p.status, 4)) { ok = false; break; }
      if (!mbar_wait(&bars->s_full[buf], (it >> 1) & 1, abort_flag, p.status, 4)) { ok = false; break; }
      tc_fence_after();
      const float* lse_s = sStat + st * 2 * BQ;
      const float* delta_s = lse_s + BQ;
      const bool edge = q0 < kb * AT + AT || q0 + BQ > len;   // some keys of this block lie after some of these queries, or some queries past the end
      const uint32_t col = buf * BQ + part * 32 + lane_off;
#pragma unroll
      for (int c = 0; c < 32; c += 16) {                    // 32 at once would take more than the 96 registers there are
        uint32_t sv[16], dv[16], pk[8], dk[8];
        tmem_ld16(tS + col + c, sv);
        tmem_ld16(tDP + col + c, dv);
        tmem_ld_wait();
#pragma unroll
        for (int t = 0; t < 16; t += 4) {
          const float4 l4 = *reinterpret_cast<const float4*>(lse_s + part * 32 + c + t);
          const float4 d4 = *reinterpret_cast<const float4*>(delta_s + part * 32 + c + t);
          const f32x2 lv[2] = {pack2(l4.x, l4.y), pack2(l4.z, l4.w)}, dl[2] = {pack2(d4.x, d4.y), pack2(d4.z, d4.w)};
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int j = t + 2 * u, q = q0 + part * 32 + c + j;
            float x0, x1, s0, s1;
            unpack2(fma2(pack2(sv[j], sv[j + 1]), nscale, lv[u]), x0, x1);         // log-sum-exp minus score
            float p0 = exp2f(-x0), p1 = exp2f(-x1);
            // the softmax scale is applied to dK once, at the end
            unpack2(mul2(pack2(p0, p1), fma2(dl[u], minus, pack2(dv[j], dv[j + 1]))), s0, s1);
            if (edge && (q < kv_idx || q >= len)) p0 = s0 = 0.f;
            if (edge && (q + 1 < kv_idx || q + 1 >= len)) p1 = s1 = 0.f;
            pk[j >> 1] = pack_bf16x2(p0, p1);
            dk[j >> 1] = pack_bf16x2(s0, s1);
          }
        }
        tmem_st8(tS + col + c / 2, pk);                     // over columns that this thread has read (packed_col)
        tmem_st8(tDP + col + c / 2, dk);
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&bars->p_ready[buf]);
    }
    if (ok && mbar_wait(&bars->acc_done, 0, abort_flag, p.status, 4)) {
      tc_fence_after();
      // groups 0 and 2 store dV, 1 and 3 dK, half of the columns each
      const long long ld = buf == 0 ? p.ld_dv : p.ld_dk;
      const int row0 = kb * AT + (warp & 3) * 32;
      __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(buf == 0 ? p.dv : p.dk) + static_cast<long long>(first + row0) * ld + hk * p.hd + part * NH * 32;
      const uint32_t t_src = (buf == 0 ? tDV : tDK) + lane_off;
      const float out_scale = buf == 0 ? 1.f : p.scale;
      uint8_t* stage = smem + (warp - 2) * (NH * 2048);     // over K and V: every product has been computed
#pragma unroll 1
      for (int c = 0; c < NH; ++c) {
        uint32_t v[32];
        tmem_ld32(t_src + (part * NH + c) * 32, v);
        tmem_ld_wait();
        stage_head32<4 * NH>(stage, lane, c, v, out_scale);
      }
      store_staged<4 * NH>(dst, ld, stage, lane, len - row0, p.hd - part * NH * 32);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ================================================================================================ backward: dQ
// CTA = (query block of 128 positions, head, batch).  Q_i and dO_i stay in shared memory; K and V stream through in
// sub-blocks of 64 positions.  S = Q K^T and dP = dO V^T land in one of two TMEM buffer pairs; the softmax threads
// (two per query row) write dS as bf16 over half of the dP buffer's columns, which are then the tensor-memory
// A operand of dQ += dS K.  Also produces delta = rowsum(O * dO) for the dK/dV pass.
// TMEM: S buffers at 0 and 64, dP buffers at 128 and 192, dQ at 256.
struct DqBars {
  uint64_t qd_full, kv_full[NST], kv_empty[NST], s_full[2], p_ready[2], acc_done;
  uint32_t tmem_slot;
  int abort_flag;
  float delta[AT];
};

template <int NH>
__global__ void __launch_bounds__(BWD_THREADS, 1)
packed_dq_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                      const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmDO, PackedDev p) {
  constexpr uint32_t TILE_BYTES = NH * HALF_BYTES, Q_TILE = NH * Q_HALF;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_up_1024(smem_raw);
  uint8_t* sQ = smem;
  uint8_t* sDO = smem + TILE_BYTES;
  uint8_t* sK = smem + 2 * TILE_BYTES;                 // NST x 16 KB
  uint8_t* sV = sK + NST * Q_TILE;                     // NST x 16 KB
  uint8_t* sTerm = sV + NST * Q_TILE;                  // what delta is summed from, 16 bytes for each 8 columns of a row
  DqBars* bars = reinterpret_cast<DqBars*>(sTerm + TILE_BYTES);
  volatile int* abort_flag = &bars->abort_flag;

  const int warp = warp_id(), lane = threadIdx.x & 31;
  const int order = blockIdx.x / p.Hq, h = blockIdx.x - order * p.Hq;
  const PackedTile tile = p.tiles[order];
  const int qb = tile.index, len = tile.len, first = tile.first;
  const int hk = h / (p.Hq / p.Hkv);
  int nkv = (qb + 1) * (AT / BQ);                      // KV sub-blocks up to and including the diagonal
  const int nkv_all = (len + BQ - 1) / BQ;
  if (nkv > nkv_all) nkv = nkv_all;

  auto load_stage = [&](int j, uint32_t e) {
    const int st = j % NST;
    mbar_expect_tx(&bars->kv_full[st], 2 * Q_TILE, e);
    load_head_tile<NH>(sK + st * Q_TILE, Q_HALF, &tmK, &bars->kv_full[st], hk, first + j * BQ, 0, e);
    load_head_tile<NH>(sV + st * Q_TILE, Q_HALF, &tmV, &bars->kv_full[st], hk, first + j * BQ, 0, e);
  };
  if (warp == 0) {                     // the first loads are on their way while the block sets itself up
    if (lane == 0) {
      mbar_init(&bars->qd_full, 1);
      for (int i = 0; i < NST; ++i) { mbar_init(&bars->kv_full[i], 1); mbar_init(&bars->kv_empty[i], 1); }
      for (int i = 0; i < 2; ++i) { mbar_init(&bars->s_full[i], 1); mbar_init(&bars->p_ready[i], 256); }
      mbar_init(&bars->acc_done, 1);
      bars->abort_flag = 0;
      mbar_fence_init();
    }
    __syncwarp();
    const uint32_t e = elect_one();
    mbar_expect_tx(&bars->qd_full, 2 * TILE_BYTES, e);
    load_head_tile<NH>(sQ, HALF_BYTES, &tmQ, &bars->qd_full, h, first + qb * AT, 0, e);
    load_head_tile<NH>(sDO, HALF_BYTES, &tmDO, &bars->qd_full, h, first + qb * AT, 0, e);
    for (int j = 0; j < NST && j < nkv; ++j) load_stage(j, e);
  }
  // delta = sum over the head of o * dO.  The 16 warps take 8 rows of o each, LPR lanes to a row, and find dO in shared memory
  // later.  One thread to a row, reading both rows 16 bytes at a time, took 9000 of the 50000 cycles of the longest block.
  // What one thread to a row still does is the sum, from shared memory: pairs of columns, first to last, so that delta is the
  // same for every split of the loads.  (Summed over the lanes instead, its last bit moved one dS in some thousand across a
  // bf16 boundary.)
  constexpr int LPR = 8 * NH, PASSES = LPR / 4;
  uint4 o4[PASSES];
  if (warp >= 2) {
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int r = qb * AT + (warp - 2) * 8 + (i * 32 + lane) / LPR, c = (lane % LPR) * 8;
      o4[i] = make_uint4(0, 0, 0, 0);
      if (r < len && c < p.hd)
        o4[i] = *reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(p.o_in) + static_cast<long long>(first + r) * p.ld_o + h * p.hd + c);
    }
  }
  if (warp == 1) tmem_alloc(&bars->tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, bars->tmem_slot, 0);
  const uint32_t tS = tmem, tDP = tmem + 128, tDQ = tmem + 256;

  if (warp == 0) {
    const uint32_t e = elect_one();
    for (int j = NST; j < nkv; ++j) {
      if (!mbar_wait_warp(&bars->kv_empty[j % NST], ((j / NST) & 1) ^ 1, abort_flag, p.status, 4)) break;
      load_stage(j, e);
    }
  } else if (warp == 1) {
    {
      const uint32_t e = elect_one();
      constexpr uint32_t idesc_s = umma_idesc_bf16(128, BQ, false, false);
      constexpr uint32_t idesc_acc = umma_idesc_bf16(128, 64 * NH, false, true);
      const uint64_t q_desc = kmajor_desc(sQ), do_desc = kmajor_desc(sDO), k_desc = kmajor_desc(sK), v_desc = kmajor_desc(sV);
      const uint64_t k_mn = mnmajor_desc(sK, Q_HALF);
      bool ok = mbar_wait_warp(&bars->qd_full, 0, abort_flag, p.status, 4);
      auto issue_sp = [&](int j) -> bool {
        const int st = j % NST, buf = j & 1;
        if (!mbar_wait_warp(&bars->kv_full[st], (j / NST) & 1, abort_flag, p.status, 4)) return false;
        if ((j + 1) * BQ > len) clear_rows<NH>(sK + st * Q_TILE, Q_HALF, len - j * BQ, BQ, lane);
        tc_fence_after();
#pragma unroll
        for (int ks = 0; ks < 4 * NH; ++ks)
          umma_ss(tS + buf * BQ, desc_at(q_desc, kmajor_off(HALF_BYTES, ks)), desc_at(k_desc, st * Q_TILE + kmajor_off(Q_HALF, ks)), idesc_s, ks > 0 ? 1u : 0u, e);
#pragma unroll
        for (int ks = 0; ks < 4 * NH; ++ks)
          umma_ss(tDP + buf * BQ, desc_at(do_desc, kmajor_off(HALF_BYTES, ks)), desc_at(v_desc, st * Q_TILE + kmajor_off(Q_HALF, ks)), idesc_s, ks > 0 ? 1u : 0u, e);
        umma_commit(&bars->s_full[buf], e);
        return true;
      };
      if (ok) ok = issue_sp(0);
      for (int j = 0; ok && j < nkv; ++j) {
        if (j + 1 < nkv) { ok = issue_sp(j + 1); if (!ok) break; }
        const int st = j % NST, buf = j & 1;
        if (!mbar_wait_warp(&bars->p_ready[buf], (j >> 1) & 1, abort_flag, p.status, 4)) break;
        tc_fence_after();
#pragma unroll
        for (int ks = 0; ks < BQ / 16; ++ks)
          umma_ts(tDQ, tDP + buf * BQ + packed_col(ks), desc_at(k_mn, st * Q_TILE + mnmajor_off(ks)), idesc_acc, (j > 0 || ks > 0) ? 1u : 0u, e);
        umma_commit(&bars->kv_empty[st], e);
      }
      if (ok) umma_commit(&bars->acc_done, e);
    }
  } else {
    const int wg = (warp - 2) >> 2, buf = wg & 1, part = wg >> 1;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const int q_idx = qb * AT + row;
    const long long stat_idx = h * p.stat_rows + tile.slot * AT + row;
    const float lse2 = p.lse[stat_idx];
    bool ok = mbar_wait(&bars->qd_full, 0, abort_flag, p.status, 4);
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int r = (warp - 2) * 8 + (i * 32 + lane) / LPR, c = lane % LPR;
      const uint4 g4 = *reinterpret_cast<const uint4*>(sDO + (c >> 3) * HALF_BYTES + r * 128 + (((c & 7) ^ (r & 7)) << 4));
      const uint32_t ow[4] = {o4[i].x, o4[i].y, o4[i].z, o4[i].w}, gw[4] = {g4.x, g4.y, g4.z, g4.w};
      float t[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) t[q] = bf16_lo(ow[q]) * bf16_lo(gw[q]) + bf16_hi(ow[q]) * bf16_hi(gw[q]);
      *reinterpret_cast<float4*>(sTerm + staged_at<LPR>(r, c)) = make_float4(t[0], t[1], t[2], t[3]);
    }
    named_barrier(1, 512);                                // all groups: the terms are in shared memory
    if (wg == 0) {
      float d = 0.f;
#pragma unroll
      for (int c = 0; c < LPR; ++c) {
        const float4 t = *reinterpret_cast<const float4*>(sTerm + staged_at<LPR>(row, c));
        d += t.x; d += t.y; d += t.z; d += t.w;
      }
      bars->delta[row] = d;
      p.delta[stat_idx] = d;
    }
    named_barrier(1, 512);                                // and the block's delta values
    const float delta = bars->delta[row];
    const f32x2 nscale = pack2(-p.scale_log2, -p.scale_log2), lse_2 = pack2(lse2, lse2), ndelta = pack2(-delta, -delta);
    for (int j = buf; ok && j < nkv; j += 2) {
      if (!mbar_wait(&bars->s_full[buf], (j >> 1) & 1, abort_flag, p.status, 4)) { ok = false; break; }
      tc_fence_after();
      const int kv0 = j * BQ;
      const bool diag = (kv0 + BQ - 1 > qb * AT);
      const uint32_t col = buf * BQ + part * 32 + lane_off;
      uint32_t sv[32], dv[32];
      tmem_ld32(tS + col, sv);
      tmem_ld32(tDP + col, dv);
      tmem_ld_wait();
      uint32_t dk[16];
#pragma unroll
      for (int t = 0; t < 32; t += 2) {
        float x0, x1, s0, s1;
        unpack2(fma2(pack2(sv[t], sv[t + 1]), nscale, lse_2), x0, x1);             // log-sum-exp minus score
        float p0 = exp2f(-x0), p1 = exp2f(-x1);
        unpack2(mul2(pack2(p0, p1), add2(pack2(dv[t], dv[t + 1]), ndelta)), s0, s1);
        if (diag && (kv0 + part * 32 + t > q_idx)) s0 = 0.f;
        if (diag && (kv0 + part * 32 + t + 1 > q_idx)) s1 = 0.f;
        dk[t >> 1] = pack_bf16x2(s0, s1);
      }
      tmem_st16(tDP + col, dk);                             // over columns that this thread has read (packed_col)
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&bars->p_ready[buf]);
    }
    if (ok && mbar_wait(&bars->acc_done, 0, abort_flag, p.status, 4)) {
      tc_fence_after();
      // the groups store 32 dQ columns each (two of them where the head is one half wide); dS was left unscaled, so the
      // softmax scale lands here
      if (wg < 2 * NH) {
        const int row0 = qb * AT + (warp & 3) * 32;
        uint8_t* stage = smem + (warp - 2) * 2048;          // over Q and dO: every product has been computed
        uint32_t v[32];
        tmem_ld32(tDQ + lane_off + wg * 32, v);
        tmem_ld_wait();
        stage_head32<4>(stage, lane, 0, v, p.scale);
        store_staged<4>(reinterpret_cast<__nv_bfloat16*>(p.dq) + static_cast<long long>(first + row0) * p.ld_dq + h * p.hd + wg * 32,
                        p.ld_dq, stage, lane, len - row0, p.hd - wg * 32);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace

// ================================================================================================ host
static void check(const PackedAttnArgs& a) {
  if (a.Hq <= 0 || a.Hkv <= 0 || a.Hq % a.Hkv || a.rows <= 0 || a.n_tiles < 0) throw std::runtime_error("himuon packed attention: bad sizes");
  if (a.hd <= 0 || a.hd > 128 || a.hd % 8) throw std::runtime_error("himuon packed attention: head_dim must be a multiple of 8 up to 128");
  if (static_cast<long long>(a.n_tiles) * a.Hq >= (1LL << 31)) throw std::runtime_error("himuon packed attention: too many tiles for one launch");
}
static PackedDev make_dev(const PackedAttnArgs& a) {
  PackedDev p{};
  p.o = a.o; p.o_in = a.o; p.lse = a.lse; p.delta = a.delta; p.dq = a.dq; p.dk = a.dk; p.dv = a.dv;
  p.Hq = a.Hq; p.Hkv = a.Hkv; p.hd = a.hd;
  p.stat_rows = static_cast<long long>(a.n_tiles) * AT;
  p.ld_o = a.ld_o; p.ld_dq = a.ld_dq; p.ld_dk = a.ld_dk; p.ld_dv = a.ld_dv;
  p.scale = a.scale; p.scale_log2 = a.scale * kLog2e;
  p.status = status_word_ptr();
  return p;
}
template <typename K>
static void allow_smem(K kern, size_t bytes) {
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  if (e != cudaSuccess) throw std::runtime_error(std::string("himuon packed attention: ") + cudaGetErrorString(e));
}
static void check_launch(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) throw std::runtime_error(std::string("himuon packed attention ") + what + " launch failed: " + cudaGetErrorString(e));
}

template <int NH>
static void launch_fwd(const PackedAttnArgs& a, cudaStream_t s) {
  constexpr size_t SMEM = 1024 + NH * HALF_BYTES + 4 * NH * KV_HALF + 256;
  allow_smem(packed_fwd_kernel<NH>, SMEM);
  PackedDev p = make_dev(a);
  p.tiles = a.by_keys;
  const CUtensorMap tq = head_tmap(a.q, 1, a.rows, a.Hq, a.hd, a.ld_q), tk = head_tmap(a.k, 1, a.rows, a.Hkv, a.hd, a.ld_k, BKV),
                    tv = head_tmap(a.v, 1, a.rows, a.Hkv, a.hd, a.ld_v, BKV);
  packed_fwd_kernel<NH><<<a.n_tiles * a.Hq, 192, SMEM, s>>>(tq, tk, tv, p);
}
void packed_attn_fwd(const PackedAttnArgs& a, cudaStream_t s) {
  check(a);
  if (a.n_tiles == 0) return;
  if (head_halves(a.hd) == 1) launch_fwd<1>(a, s);
  else launch_fwd<2>(a, s);
  check_launch("forward");
}

template <int NH>
static void launch_bwd(const PackedAttnArgs& a, cudaStream_t s) {
  constexpr size_t SMEM_KV = 1024 + 2 * NH * HALF_BYTES + 2 * NST * NH * Q_HALF + NST * STAT_BYTES + sizeof(DkvBars) + 64;
  constexpr size_t SMEM_Q = 1024 + 3 * NH * HALF_BYTES + 2 * NST * NH * Q_HALF + sizeof(DqBars) + 64;
  static_assert(SMEM_KV <= 232448 && SMEM_Q <= 232448, "shared memory budget of one CTA exceeded");
  allow_smem(packed_dkv_kernel<NH>, SMEM_KV);
  allow_smem(packed_dq_kernel<NH>, SMEM_Q);
  PackedDev p = make_dev(a);
  const CUtensorMap tq = head_tmap(a.q, 1, a.rows, a.Hq, a.hd, a.ld_q), tdo = head_tmap(a.d_o, 1, a.rows, a.Hq, a.hd, a.ld_do),
                    tk = head_tmap(a.k, 1, a.rows, a.Hkv, a.hd, a.ld_k), tv = head_tmap(a.v, 1, a.rows, a.Hkv, a.hd, a.ld_v),
                    tq64 = head_tmap(a.q, 1, a.rows, a.Hq, a.hd, a.ld_q, BQ), tdo64 = head_tmap(a.d_o, 1, a.rows, a.Hq, a.hd, a.ld_do, BQ),
                    tk64 = head_tmap(a.k, 1, a.rows, a.Hkv, a.hd, a.ld_k, BQ), tv64 = head_tmap(a.v, 1, a.rows, a.Hkv, a.hd, a.ld_v, BQ);
  p.tiles = a.by_keys;
  packed_dq_kernel<NH><<<a.n_tiles * a.Hq, BWD_THREADS, SMEM_Q, s>>>(tq, tk64, tv64, tdo, p);      // and delta, which the other reads
  check_launch("dQ");
  p.tiles = a.by_queries;
  packed_dkv_kernel<NH><<<a.n_tiles * a.Hkv, BWD_THREADS, SMEM_KV, s>>>(tq64, tk, tv, tdo64, p);
  check_launch("dK / dV");
}
void packed_attn_bwd(const PackedAttnArgs& a, cudaStream_t s) {
  check(a);
  if (a.n_tiles == 0) return;
  if (head_halves(a.hd) == 1) launch_bwd<1>(a, s);
  else launch_bwd<2>(a, s);
}

}  // namespace himuon
