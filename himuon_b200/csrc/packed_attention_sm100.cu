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
#include "packed_attention.cuh"

namespace himuon {

namespace {

// ================================================================================================ forward
// One block per SM, over a list of items; an item is two tiles of 128 queries that read the same keys: two query heads of one KV head,
// or, where a KV head has an odd number of them, two neighbouring tiles of one head (the second has more keys, or is not there).
// K and V come in blocks of 64 positions through a ring.  Tensor memory: two S buffers for each tile, at 0, 64 and 128, 192 (P, bf16,
// over the first 32 columns of its S), O at 256 and 384.
// Each tile has four warps, one thread a row.  The next Q K^T of a tile is issued ahead of the P V that its warps still work for, so
// that they find scores when they are done.  Probabilities are taken relative to an older maximum of the row, and only where it has grown
// by more than 2^8 (in base-2 units) is O rescaled.  The block's loads run ahead of its products across items; O leaves by TMA.
//
// Measured, one document of 8192 tokens, 32 heads over 8 of 128: 440 us, 1250 TFLOP/s (one tile a block, two blocks per SM, 580; blocks of 128
// keys with one S a tile, where scores, probabilities, P V and the next scores follow one another, 501).  A step of 64 keys took 1650
// cycles without the sums of rounded weights (435 us).  Its products alone take 1239 (products of 128 x 64 x 16 with both operands in shared memory 48, those of P V 64 each), and
// shared memory is busy for 1280 of them: the operands, and 32 KB of new K and V.  What the issuing warp does beside issuing counts in full,
// because an MMA is issued about when it starts (the tensor core keeps two more): with a general step, ring positions found by division and
// item fields that are not uniform the same step took 2200.  24 documents of 341 tokens in the mean, 16 heads over 8: 57 us, where an item has
// some nine steps and 4300 cycles for its first scores, its last product and its epilogue.  What a backward pass needs (KEEP) costs 3 us there, 22 at the
// one document (in a training step; 60 where this kernel alone runs, at the power limit).
constexpr int FWD_THREADS = 320;                     // warps 0-3 and 4-7: rows of the tiles, 8: TMA, 9: MMA
constexpr int BKV = 64;                              // key positions per block
constexpr uint32_t KV_HALF = BKV * 128;              // one 64-column half of a K or V block: 8 KB
constexpr int FWD_SLOTS = 6;
struct FwdBars {
  uint64_t q_full[2], q_empty[2], kv_full[FWD_SLOTS], kv_empty[FWD_SLOTS], s_full[2][2], p_ready[2][2], o_done[2][2], acc_done[2], o_free[2];
  uint32_t tmem_slot;
  int abort_flag;
};

struct FwdItem {
  int first, len, hk, blocks;                        // blocks: key blocks of the longer tile
  int index[2], head[2], n[2];                       // tile number in the document, head, key blocks (0: no such tile)
  int slot[2];                                       // of the statistics
};
__device__ __forceinline__ FwdItem fwd_item(const PackedDev& p, int i) {
  FwdItem it;
  const int per = p.pair_heads ? p.Hq / 2 : p.Hq, order = i / per, y = i - order * per;
  const PackedTile t = p.tiles[order];
  it.first = t.first;
  it.len = t.len;
  it.head[0] = p.pair_heads ? 2 * y : y;
  it.head[1] = it.head[0] + p.pair_heads;
  it.hk = it.head[0] / (p.Hq / p.Hkv);
  it.index[0] = t.index;
  it.index[1] = t.index + 1 - p.pair_heads;
  it.slot[0] = t.slot;
  it.slot[1] = t.slot + 1 - p.pair_heads;
  const int all = (t.len + BKV - 1) / BKV;           // key blocks up to and including the diagonal
  it.n[0] = min((t.index + 1) * (AT / BKV), all);
  it.n[1] = it.index[1] * AT < t.len ? min((it.index[1] + 1) * (AT / BKV), all) : 0;
  it.blocks = it.n[0] > it.n[1] ? it.n[0] : it.n[1];
  return it;
}
__device__ __forceinline__ FwdItem fwd_item_uniform(const PackedDev& p, int i) {
  FwdItem it = fwd_item(p, i);
  it.first = uniform(it.first); it.len = uniform(it.len); it.hk = uniform(it.hk); it.blocks = uniform(it.blocks);
#pragma unroll
  for (int t = 0; t < 2; ++t) { it.index[t] = uniform(it.index[t]); it.head[t] = uniform(it.head[t]); it.n[t] = uniform(it.n[t]); }
  return it;
}
// What the warps of tile t need of it.
struct FwdRow { int first, len, index, head, n, slot; };
__device__ __forceinline__ FwdRow fwd_row(const PackedDev& p, int i, int t) {
  const FwdItem it = fwd_item(p, i);
  return t ? FwdRow{it.first, it.len, it.index[1], it.head[1], it.n[1], it.slot[1]} : FwdRow{it.first, it.len, it.index[0], it.head[0], it.n[0], it.slot[0]};
}
// e^(scaled score - maximum) of 32 scores as bf16, and the sums of what was not rounded yet.  (A part of the exponentials as polynomials on the FMA units only costs:
// 447 us for one document of 8192 tokens without, 448, 465 and 492 with an eighth, three and five eighths.)
template <bool SUM>
__device__ __forceinline__ void to_probabilities(const uint32_t (&v)[32], f32x2 scale2, f32x2 m2, f32x2 (&sum)[2], uint32_t (&pk)[16]) {
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    float p0, p1;
    unpack2(fma2(pack2(v[2 * k], v[2 * k + 1]), scale2, m2), p0, p1);
    p0 = exp2f(p0);                                  // (of a masked score, -inf, 0)
    p1 = exp2f(p1);
    if (SUM) sum[k & 1] = add2(sum[k & 1], pack2(p0, p1));
    pk[k] = pack_bf16x2(p0, p1);
  }
}
// Sums of the rounded ones.  O is divided by these: its weights then add up to 1, and a row with one weight near 1 keeps what delta has beside it.
// (Divided by the others O is off by up to 2^-8 of that one's V where its weight is relative to an older maximum: gradients of rows with 1e-3 to 1e-2 beside a
// weight were off by 4 to 6 % in documents of 700 to 2000 tokens, of others by 0.25.)  An addition takes a bf16 as it is: 2 instructions a pair for 3 with
// shifts and packed sums, 447 us for 455 over five documents of 16384 tokens, 439 with the unrounded sums, which the exponentials hide better.
__device__ __forceinline__ void add_rounded(const uint32_t (&pk)[16], float (&sum)[4]) {
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const unsigned short lo = static_cast<unsigned short>(pk[k]), hi = static_cast<unsigned short>(pk[k] >> 16);
    asm("add.f32.bf16 %0, %1, %0;" : "+f"(sum[(2 * k) & 3]) : "h"(lo));
    asm("add.f32.bf16 %0, %1, %0;" : "+f"(sum[(2 * k + 1) & 3]) : "h"(hi));
  }
}
__device__ __forceinline__ float total(const f32x2 (&sum)[2]) {
  float s0, s1;
  unpack2(add2(sum[0], sum[1]), s0, s1);
  return s0 + s1;
}
__device__ __forceinline__ float largest32(const uint32_t (&v)[32]) {
  float a = __uint_as_float(v[0]), b = __uint_as_float(v[1]);
#pragma unroll
  for (int k = 2; k + 3 < 32; k += 4) {
    a = max3(a, __uint_as_float(v[k]), __uint_as_float(v[k + 1]));
    b = max3(b, __uint_as_float(v[k + 2]), __uint_as_float(v[k + 3]));
  }
  return max3(fmaxf(a, b), __uint_as_float(v[30]), __uint_as_float(v[31]));
}
// -inf for keys behind the row's own token: key0 + k > row.
__device__ __forceinline__ void mask_future(uint32_t (&v)[32], int key0, int row) {
#pragma unroll
  for (int k = 0; k < 32; ++k) v[k] = key0 + k > row ? 0xFF800000u : v[k];
}

// KEEP: for a backward pass, with the log-sum-exps and O's low bits.
template <int NH, bool KEEP>
__global__ void __launch_bounds__(FWD_THREADS, 1)
packed_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const __grid_constant__ CUtensorMap tmO, PackedDev p) {
  constexpr uint32_t TILE_BYTES = NH * HALF_BYTES, KV_TILE = NH * KV_HALF;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_up_1024(smem_raw);
  uint8_t* sQ = smem;                                // two tiles
  uint8_t* sKV = smem + 2 * TILE_BYTES;              // the ring
  uint8_t* sOut = sKV + FWD_SLOTS * KV_TILE;         // for each of eight warps 32 rows of O, halves of 64 columns
  FwdBars* bars = reinterpret_cast<FwdBars*>(sOut + 8 * NH * 4096);
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = warp_id(), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&bars->q_full[t], 1); mbar_init(&bars->q_empty[t], 1);
      for (int b = 0; b < 2; ++b) { mbar_init(&bars->s_full[t][b], 1); mbar_init(&bars->p_ready[t][b], 128); mbar_init(&bars->o_done[t][b], 1); }
      mbar_init(&bars->acc_done[t], 1); mbar_init(&bars->o_free[t], 128);
    }
    for (int i = 0; i < FWD_SLOTS; ++i) { mbar_init(&bars->kv_full[i], 1); mbar_init(&bars->kv_empty[i], 1); }
    bars->abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 9) tmem_alloc(&bars->tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, bars->tmem_slot, 0);

  if (warp == 8) {
    // ------------------------------------------------------------ TMA
    const uint32_t e = elect_one();
    int used[2] = {0, 0}, kv = 0;
    bool ok = true;
    auto load_kv = [&](const CUtensorMap* tm, const FwdItem& it, int j) {
      const int s = kv % FWD_SLOTS;
      if (!mbar_wait_warp(&bars->kv_empty[s], ((kv / FWD_SLOTS) & 1) ^ 1, abort_flag, p.status, 4)) return false;
      mbar_expect_tx(&bars->kv_full[s], KV_TILE, e);
      load_head_tile<NH>(sKV + s * KV_TILE, KV_HALF, tm, &bars->kv_full[s], it.hk, it.first + j * BKV, 0, e);
      ++kv;
      return true;
    };
    for (int round = 0, i; ok && (i = my_turn(round)) < p.n_items; ++round) {
      const FwdItem it = fwd_item_uniform(p, i);
      ok = load_kv(&tmK, it, 0);                     // (ahead of Q, which waits for the item before to be done with its own)
      for (int t = 0; ok && t < 2; ++t) {
        if (it.n[t] == 0) continue;
        ok = mbar_wait_warp(&bars->q_empty[t], (used[t] & 1) ^ 1, abort_flag, p.status, 4);
        if (!ok) break;
        mbar_expect_tx(&bars->q_full[t], TILE_BYTES, e);
        load_head_tile<NH>(sQ + t * TILE_BYTES, HALF_BYTES, &tmQ, &bars->q_full[t], it.head[t], it.first + it.index[t] * AT, 0, e);
        ++used[t];
      }
      ok = ok && load_kv(&tmV, it, 0);
      for (int j = 1; ok && j < it.blocks; ++j) ok = load_kv(&tmK, it, j) && load_kv(&tmV, it, j);
    }
  } else if (warp == 9) {
    // ------------------------------------------------------------ MMA issue
    const uint32_t e = elect_one();
    constexpr uint32_t idesc_s = umma_idesc_bf16(128, BKV, false, false);
    constexpr uint32_t idesc_pv = umma_idesc_bf16(128, 64 * NH, false, true);
    const uint64_t q_desc = kmajor_desc(sQ), k_desc = kmajor_desc(sKV), v_desc = mnmajor_desc(sKV, KV_HALF);
    // An MMA is issued about when it starts: the tensor core has work for two more, some 128 cycles.  A wait for a barrier costs that long even
    // if its phase is over, so the next one is looked at before the last products ahead of it are issued.
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity, bool there) { ok = ok && (there || mbar_wait_warp(bar, parity, abort_flag, p.status, 4)); };
    // Where a step's K (slot 2c) and V (slot 2c + 1) are in the ring: kept, because finding it anew for every use takes longer than a product.
    struct Place {
      uint32_t c, parity;
      __device__ __forceinline__ Place next() const { return c == FWD_SLOTS / 2 - 1 ? Place{0, parity ^ 1} : Place{c + 1, parity}; }
    };
    Place here{0, 0};
    uint32_t scored[2] = {0, 0}, summed[2] = {0, 0}, items[2] = {0, 0};
    // Products `from` to `to` of the 4 NH of Q K^T of tile t, into the S buffer that P V of the last step but one has been issued for.
    auto issue_s = [&](auto tile, uint32_t k_off, int from, int to) {
      constexpr int t = decltype(tile)::value;
      const uint32_t d = tmem + t * 128 + (scored[t] & 1) * BKV;
      const uint64_t kd = desc_at(k_desc, k_off);
#pragma unroll
      for (int ks = 0; ks < 4 * NH; ++ks)
        if (ks >= from && ks < to) umma_ss(d, desc_at(q_desc, t * TILE_BYTES + kmajor_off(HALF_BYTES, ks)), desc_at(kd, kmajor_off(KV_HALF, ks)), idesc_s, ks > 0 ? 1u : 0u, e);
    };
    auto done_s = [&](auto tile, bool last) {        // `last`: the last one that needs its Q
      constexpr int t = decltype(tile)::value;
      umma_commit(&bars->s_full[t][scored[t]++ & 1], e);
      if (last) umma_commit(&bars->q_empty[t], e);
    };
    auto first_s = [&](auto tile, const FwdItem& it, const Place& at) {
      constexpr int t = decltype(tile)::value;
      if (!ok || it.n[t] == 0) return;
      wait(&bars->q_full[t], items[t] & 1, false);
      wait(&bars->kv_full[2 * at.c], at.parity, false);
      if (!ok) return;
      tc_fence_after();
      issue_s(tile, at.c * 2 * KV_TILE, 0, 4 * NH);
      done_s(tile, it.n[t] == 1);
    };
    const std::integral_constant<int, 0> T0;
    const std::integral_constant<int, 1> T1;
    int i = my_turn(0);
    FwdItem it{};
    if (i < p.n_items) {
      it = fwd_item_uniform(p, i);
      first_s(T0, it, here);
      first_s(T1, it, here);
      if (ok) umma_commit(&bars->kv_empty[0], e);
    }
    for (int round = 0; ok && i < p.n_items; ++round) {
      const int i_next = my_turn(round + 1);
      FwdItem next{};
      if (i_next < p.n_items) next = fwd_item_uniform(p, i_next);
      bool k_there = false;                          // of the next block
      // A step; `inner`: neither the first nor the last or last but one of a tile, for which nothing has to be asked.
      auto step = [&](int j, auto inner) {
        constexpr bool IN = decltype(inner)::value;
        const Place then = here.next();
        const uint32_t v_off = here.c * 2 * KV_TILE + KV_TILE, k_off = then.c * 2 * KV_TILE;
        uint64_t *v_full = &bars->kv_full[2 * here.c + 1], *k_full = &bars->kv_full[2 * then.c];
        const uint64_t vd = desc_at(v_desc, v_off);
        const bool more = IN || j + 1 < it.blocks;
        bool v_there = false;
        if (more) wait(k_full, then.parity, k_there);
        k_there = false;
        if (!ok) return;
        tc_fence_after();
        auto turn = [&](auto tile) {
          constexpr int t = decltype(tile)::value;
          const uint32_t b = summed[t] & 1, p_par = (summed[t] >> 1) & 1;
          uint64_t* p_bar = &bars->p_ready[t][b];
          bool p_there = false;
          if (IN || j + 1 < it.n[t]) {
            issue_s(tile, k_off, 0, 4 * NH - 2);
            p_there = mbar_peek(p_bar, p_par);
            if (t == 0) v_there = mbar_peek(v_full, here.parity);
            issue_s(tile, k_off, 4 * NH - 2, 4 * NH);
            done_s(tile, !IN && j + 2 == it.n[t]);
          }
          if (t == 1 && more) umma_commit(&bars->kv_empty[2 * then.c], e);
          if (t == 0) {
            wait(v_full, here.parity, v_there);
            if (!IN && ok && (j + 1) * BKV > it.len) clear_rows<NH>(sKV + v_off, KV_HALF, it.len - j * BKV, BKV, lane);
          }
          if (!IN && j >= it.n[t]) return;
          if (!IN && j == 0) wait(&bars->o_free[t], (items[t] & 1) ^ 1, false);
          wait(p_bar, p_par, p_there);
          if (!ok) return;
          ++summed[t];
          tc_fence_after();
          const uint32_t tP = tmem + t * 128 + b * BKV;
#pragma unroll
          for (int ks = 0; ks < BKV / 16; ++ks) {
            if (t == 1 && ks == BKV / 16 - 1 && (IN || j + 2 < it.blocks)) {
              const Place after = then.next();
              k_there = mbar_peek(&bars->kv_full[2 * after.c], after.parity);
            }
            umma_ts(tmem + 256 + t * 128, tP + ks * 8, desc_at(vd, mnmajor_off(ks)), idesc_pv, (IN || j > 0 || ks > 0) ? 1u : 0u, e);
          }
          umma_commit(&bars->o_done[t][b], e);
          if (!IN && j + 1 == it.n[t]) {
            umma_commit(&bars->acc_done[t], e);
            ++items[t];
          }
        };
        turn(T0);
        turn(T1);
        if (!ok) return;
        umma_commit(&bars->kv_empty[2 * here.c + 1], e);
        here = then;
      };
      const int inner_end = (it.n[0] < it.n[1] ? it.n[0] : it.n[1]) - 2;      // first step that is no inner one
      int j = 0;
      step(j++, std::false_type{});
      for (; ok && j < inner_end; ++j) step(j, std::true_type{});
      for (; ok && j < it.blocks; ++j) step(j, std::false_type{});
      if (next.blocks > 0) {
        first_s(T0, next, here);
        first_s(T1, next, here);
        if (ok) umma_commit(&bars->kv_empty[2 * here.c], e);
      }
      it = next;
      i = i_next;
    }
  } else {
    // ------------------------------------------------------------ softmax and epilogue: one thread per query row
    const int t = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS0 = tmem + t * 128 + lane_off, tO = tmem + 256 + t * 128 + lane_off;
    uint8_t* stage = sOut + warp * NH * 4096;
    zero_padding(p.o, p.ld_o, p.tokens, p.rows, p.Hq * p.hd, threadIdx.x, 256);
    const f32x2 scale2 = pack2(p.scale_log2, p.scale_log2);
    int steps = 0, items = 0;
    bool ok = true;
    auto my_item = [&](int i) { return i < p.n_items ? fwd_row(p, i, t) : FwdRow{}; };
    FwdRow it = my_item(my_turn(0));
    for (int round = 0; ok && it.len > 0; ++round) {
      const FwdRow next = my_item(my_turn(round + 1));      // (looked up early)
      const int n = it.n, diag0 = it.index * (AT / BKV);
      if (n == 0) { it = next; continue; }
      float m = -INFINITY, l = 0.f, l_rounded = 0.f;      // (l only where the log-sum-exps are kept)
      for (int j = 0; j < n; ++j, ++steps) {
        const int b = steps & 1;
        if (!mbar_wait(&bars->s_full[t][b], (steps >> 1) & 1, abort_flag, p.status, 4)) { ok = false; break; }
        tc_fence_after();
        const uint32_t tS = tS0 + b * BKV;
        const bool diag = j >= diag0;
        uint32_t v[2][32], pk[2][16];
        tmem_ld32(tS, v[0]);
        tmem_ld32(tS + 32, v[1]);
        tmem_ld_wait();
        if (diag) {
          mask_future(v[0], (j - diag0) * BKV, row);
          mask_future(v[1], (j - diag0) * BKV + 32, row);
        }
        const float m_new = fmaxf(m, fmaxf(largest32(v[0]), largest32(v[1])) * p.scale_log2);
        if (j == 0) {
          m = m_new;
        } else if (__any_sync(0xffffffffu, m_new - m > 8.f)) {
          // O (and l) move to the new maximum: the P V before this step has to be in O first
          if (!mbar_wait(&bars->o_done[t][b ^ 1], ((steps - 1) >> 1) & 1, abort_flag, p.status, 4)) { ok = false; break; }
          tc_fence_after();
          const float alpha = exp2f(m - m_new);
          m = m_new;
#pragma unroll 1
          for (int c = 0; c < 4 * NH; ++c) {
            uint32_t o[16];
            tmem_ld16(tO + c * 16, o);
            tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
            tmem_st16(tO + c * 16, o);
          }
          l *= alpha;
          l_rounded *= alpha;
        }
        const f32x2 m2 = pack2(-m, -m);
        f32x2 sum[2] = {pack2(0.f, 0.f), pack2(0.f, 0.f)};
        to_probabilities<KEEP>(v[0], scale2, m2, sum, pk[0]);
        to_probabilities<KEEP>(v[1], scale2, m2, sum, pk[1]);
        tmem_st16(tS, pk[0]);                            // over scores that are in registers
        tmem_st16(tS + 16, pk[1]);
        if (KEEP) l += total(sum);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&bars->p_ready[t][b]);
        float rounded[4] = {0.f, 0.f, 0.f, 0.f};      // (beside the product)
        add_rounded(pk[0], rounded);
        add_rounded(pk[1], rounded);
        l_rounded += (rounded[0] + rounded[1]) + (rounded[2] + rounded[3]);
      }
      if (!ok || !mbar_wait(&bars->acc_done[t], items++ & 1, abort_flag, p.status, 4)) { ok = false; break; }
      tc_fence_after();
      const float inv = 1.f / l_rounded;
      const int q0 = it.index * AT + (warp & 3) * 32, rows = it.len - q0;
      const bool whole = rows >= 32;                     // uniform over the warp
      tma_store_wait_read<0>();                          // the item before has left the buffer (whichever lane sent it)
      __syncwarp();
#pragma unroll 1
      for (int c = 0; c < 2 * NH; ++c) {
        uint32_t o[32];
        tmem_ld32(tO + c * 32, o);
        tmem_ld_wait();
        if constexpr (KEEP) {
          signed char* low = p.o_low + low_at(p, it.head, it.slot, row, c * 32);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              float f[4];
#pragma unroll
              for (int x = 0; x < 4; ++x) f[x] = __uint_as_float(o[h * 16 + k * 4 + x]) * inv;
              w[k] = low_of(f[0], f[1], f[2], f[3], pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]));
            }
            if (c * 32 + h * 16 < p.low_ld && lane < rows) *reinterpret_cast<uint4*>(low + h * 16 * AT) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        if (whole) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *reinterpret_cast<uint4*>(stage + (c >> 1) * 4096 + lane * 128 + ((((c & 1) * 4 + q) ^ (lane & 7)) << 4)) = head8(o + 8 * q, inv);
        } else if (lane < rows) {                        // the end of a document: what follows is another's
          __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(p.o) + static_cast<long long>(it.first + q0 + lane) * p.ld_o + it.head * p.hd + c * 32;
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (c * 32 + q * 8 < p.hd) *reinterpret_cast<uint4*>(out + q * 8) = head8(o + 8 * q, inv);
        }
      }
      tc_fence_before();
      mbar_arrive(&bars->o_free[t]);
      if (whole) {
        fence_proxy_async_smem();
        __syncwarp();
        const uint32_t e = elect_one();
#pragma unroll
        for (int c = 0; c < NH; ++c)
          if (c * 64 < p.hd) tma_store_4d(&tmO, stage + c * 4096, c * 64, it.head, it.first + q0, 0, e);
        if (e) tma_store_commit();
      }
      // minus the base-2 log-sum-exp of the scaled scores; rows past the end: such that their probabilities are 0
      if (KEEP) p.nlse[it.head * p.stat_rows + static_cast<long long>(it.slot) * AT + row] = lane < rows ? -m - log2f(l) : -INFINITY;
      it = next;
    }
    tma_store_wait_all();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace

// ================================================================================================ host
// 32 positions by 64 columns of a head, as the forward pass stores them.
static CUtensorMap piece_tmap(const void* ptr, int rows, int H, int hd, long long ld) {
  const uint64_t dims[4] = {static_cast<uint64_t>(hd), static_cast<uint64_t>(H), static_cast<uint64_t>(rows), 1};
  const uint64_t strides[3] = {static_cast<uint64_t>(hd) * 2, static_cast<uint64_t>(ld) * 2, static_cast<uint64_t>(ld) * 2 * static_cast<uint64_t>(rows)};
  const uint32_t box[4] = {64, 1, 32, 1};
  return make_tmap(ptr, 4, dims, strides, box, 2, true);
}

template <int NH, bool KEEP>
static void launch_fwd(const PackedAttnArgs& a, cudaStream_t s) {
  constexpr size_t SMEM = 1024 + 2 * NH * HALF_BYTES + FWD_SLOTS * NH * KV_HALF + 8 * NH * 4096 + sizeof(FwdBars);
  static_assert(SMEM <= 232448, "shared memory budget of one CTA exceeded");
  static std::atomic<uint64_t> done{0};
  allow_smem(packed_fwd_kernel<NH, KEEP>, SMEM, done);
  PackedDev p = make_dev(a);
  p.pair_heads = a.Hq / a.Hkv % 2 == 0 ? 1 : 0;
  p.tiles = p.pair_heads ? a.by_keys : a.pairs;
  p.n_items = p.pair_heads ? a.n_tiles * (a.Hq / 2) : a.n_pairs * a.Hq;
  const CUtensorMap tq = head_tmap(a.q, 1, a.rows, a.Hq, a.hd, a.ld_q), tk = head_tmap(a.k, 1, a.rows, a.Hkv, a.hd, a.ld_k, BKV),
                    tv = head_tmap(a.v, 1, a.rows, a.Hkv, a.hd, a.ld_v, BKV), to = piece_tmap(a.o, a.rows, a.Hq, a.hd, a.ld_o);
  const int grid = p.n_items < num_sms() ? p.n_items : num_sms();
  packed_fwd_kernel<NH, KEEP><<<grid, FWD_THREADS, SMEM, s>>>(tq, tk, tv, to, p);
}
void packed_attn_fwd(const PackedAttnArgs& a, cudaStream_t s) {
  check_packed(a);
  if (a.n_tiles == 0) return;
  if ((a.lse == nullptr) != (a.o_low == nullptr)) throw std::runtime_error("himuon packed attention: log-sum-exps and low bits go together");
  const bool one = head_halves(a.hd) == 1;
  if (a.lse) one ? launch_fwd<1, true>(a, s) : launch_fwd<2, true>(a, s);
  else one ? launch_fwd<1, false>(a, s) : launch_fwd<2, false>(a, s);
  check_packed_launch("forward");
}

}  // namespace himuon
