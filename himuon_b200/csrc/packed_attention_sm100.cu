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

#include <atomic>
#include <string>
#include <type_traits>

namespace himuon {

namespace {

struct PackedDev {
  const PackedTile* tiles;
  void* o; float* lse; float* delta;
  const void* o_in;
  void* dq; void* dk; void* dv;
  int Hq, Hkv, hd;
  int tokens, rows;                                  // rows from `tokens` on belong to no document
  int n_items, pair_heads;                           // forward: items; 1 where an item is one tile of two heads
  long long stat_rows;                               // rows of statistics per head: 128 for each tile
  long long ld_o, ld_dq, ld_dk, ld_dv;
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

// ================================================================================================ forward
// One block per SM, over a list of items; an item is two tiles of 128 queries that read the same keys: two query heads of one KV head,
// or, where a KV head has an odd number of them, two neighbouring tiles of one head (the second has more keys, or is not there).
// K and V come in blocks of 64 positions through a ring.  Tensor memory: two S buffers for each tile, at 0, 64 and 128, 192 (P, bf16,
// over the first 32 columns of its S), O at 256 and 384.
// Each tile has four warps, one thread a row.  The next Q K^T of a tile is issued ahead of the P V that its warps still work for, so
// that they find scores when they are done.  Probabilities are taken relative to an older maximum of the row, and only where it has grown
// by more than 2^8 (in base-2 units) is O rescaled.  The block's loads run ahead of its products across items; O leaves by TMA.
//
// Measured, one document of 8192 tokens, 32 heads over 8 of 128: 447 us, 1229 TFLOP/s (one tile a block, two blocks per SM, 580; blocks of 128
// keys with one S a tile, where scores, probabilities, P V and the next scores follow one another, 501).  A step of 64 keys takes 1650
// cycles.  Its products alone take 1239 (products of 128 x 64 x 16 with both operands in shared memory 48, those of P V 64 each), and
// shared memory is busy for 1280 of them: the operands, and 32 KB of new K and V.  What the issuing warp does beside issuing counts in full,
// because an MMA is issued about when it starts (the tensor core keeps two more): with a general step, ring positions found by division and
// item fields that are not uniform the same step took 2200.  24 documents of 341 tokens in the mean, 16 heads over 8: 58 us, where an item has
// some nine steps and 4300 cycles for its first scores, its last product and its epilogue.
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
// The same in the uniform registers of a converged warp.  (What comes from memory is not uniform to the compiler, nor is anything in a
// loop that it bounds: every operand of every MMA would be moved there.)
__device__ __forceinline__ int uniform(int x) { return static_cast<int>(__reduce_or_sync(0xffffffffu, static_cast<uint32_t>(x))); }
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
// Items are listed by falling work; the blocks take them in turns, back and forth.
__device__ __forceinline__ int fwd_turn(int round) {
  const int g = static_cast<int>(gridDim.x), b = static_cast<int>(blockIdx.x);
  return round * g + ((round & 1) ? g - 1 - b : b);
}

// Rows that belong to no document, zeroed by the threads of all blocks.
__device__ __forceinline__ void zero_padding(void* out, long long ld, int from, int to, int cols, int thread, int threads) {
  const int per_row = cols / 8;
  const long long n = static_cast<long long>(to - from) * per_row;
  for (long long i = static_cast<long long>(blockIdx.x) * threads + thread; i < n; i += static_cast<long long>(gridDim.x) * threads)
    *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(out) + (from + i / per_row) * ld + (i % per_row) * 8) = make_uint4(0, 0, 0, 0);
}

// e^(scaled score - maximum) of 32 scores as bf16, and their sums.  (A part of the exponentials as polynomials on the FMA units only costs:
// 447 us for one document of 8192 tokens without, 448, 465 and 492 with an eighth, three and five eighths.)
__device__ __forceinline__ void to_probabilities(const uint32_t (&v)[32], f32x2 scale2, f32x2 m2, f32x2 (&sum)[2], uint32_t (&pk)[16]) {
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    float p0, p1;
    unpack2(fma2(pack2(v[2 * k], v[2 * k + 1]), scale2, m2), p0, p1);
    p0 = exp2f(p0);                                  // (of a masked score, -inf, 0)
    p1 = exp2f(p1);
    sum[k & 1] = add2(sum[k & 1], pack2(p0, p1));
    pk[k] = pack_bf16x2(p0, p1);
  }
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
// -inf for keys behind the row's own token: key0 + k > row.
__device__ __forceinline__ void mask_future(uint32_t (&v)[32], int key0, int row) {
#pragma unroll
  for (int k = 0; k < 32; ++k) v[k] = key0 + k > row ? 0xFF800000u : v[k];
}

template <int NH>
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
    for (int round = 0, i; ok && (i = fwd_turn(round)) < p.n_items; ++round) {
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
    int i = fwd_turn(0);
    FwdItem it{};
    if (i < p.n_items) {
      it = fwd_item_uniform(p, i);
      first_s(T0, it, here);
      first_s(T1, it, here);
      if (ok) umma_commit(&bars->kv_empty[0], e);
    }
    for (int round = 0; ok && i < p.n_items; ++round) {
      const int i_next = fwd_turn(round + 1);
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
    FwdRow it = my_item(fwd_turn(0));
    for (int round = 0; ok && it.len > 0; ++round) {
      const FwdRow next = my_item(fwd_turn(round + 1));      // (looked up early)
      const int n = it.n, diag0 = it.index * (AT / BKV);
      if (n == 0) { it = next; continue; }
      float m = -INFINITY, l = 0.f;
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
        }
        const f32x2 m2 = pack2(-m, -m);
        f32x2 sum[2] = {pack2(0.f, 0.f), pack2(0.f, 0.f)};
        to_probabilities(v[0], scale2, m2, sum, pk[0]);
        to_probabilities(v[1], scale2, m2, sum, pk[1]);
        tmem_st16(tS, pk[0]);                            // over scores that are in registers
        tmem_st16(tS + 16, pk[1]);
        float s0, s1;
        unpack2(add2(sum[0], sum[1]), s0, s1);
        l += s0 + s1;
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&bars->p_ready[t][b]);
      }
      if (!ok || !mbar_wait(&bars->acc_done[t], items++ & 1, abort_flag, p.status, 4)) { ok = false; break; }
      tc_fence_after();
      const float inv = 1.f / l;
      const int q0 = it.index * AT + (warp & 3) * 32, rows = it.len - q0;
      const bool whole = rows >= 32;                     // uniform over the warp
      tma_store_wait_read<0>();                          // the item before has left the buffer (whichever lane sent it)
      __syncwarp();
#pragma unroll 1
      for (int c = 0; c < 2 * NH; ++c) {
        uint32_t o[32];
        tmem_ld32(tO + c * 32, o);
        tmem_ld_wait();
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
      // base-2 log-sum-exp of the scaled scores; rows past the end have none
      if (p.lse) p.lse[it.head * p.stat_rows + static_cast<long long>(it.slot) * AT + row] = lane < rows ? m + log2f(l) : INFINITY;
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

  zero_padding(p.dk, p.ld_dk, p.tokens, p.rows, p.Hkv * p.hd, threadIdx.x, BWD_THREADS);
  zero_padding(p.dv, p.ld_dv, p.tokens, p.rows, p.Hkv * p.hd, threadIdx.x, BWD_THREADS);
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

  zero_padding(p.dq, p.ld_dq, p.tokens, p.rows, p.Hq * p.hd, threadIdx.x, BWD_THREADS);
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
  p.Hq = a.Hq; p.Hkv = a.Hkv; p.hd = a.hd; p.tokens = a.tokens; p.rows = a.rows;
  p.stat_rows = static_cast<long long>(a.n_tiles) * AT;
  p.ld_o = a.ld_o; p.ld_dq = a.ld_dq; p.ld_dk = a.ld_dk; p.ld_dv = a.ld_dv;
  p.scale = a.scale; p.scale_log2 = a.scale * kLog2e;
  p.status = status_word_ptr();
  return p;
}
// Once for each kernel and device.
template <typename K>
static void allow_smem(K kern, size_t bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (bit && (done.load(std::memory_order_relaxed) & bit)) return;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  if (e != cudaSuccess) throw std::runtime_error(std::string("himuon packed attention: ") + cudaGetErrorString(e));
  done.fetch_or(bit, std::memory_order_relaxed);
}
static void check_launch(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) throw std::runtime_error(std::string("himuon packed attention ") + what + " launch failed: " + cudaGetErrorString(e));
}

// 32 positions by 64 columns of a head, as the forward pass stores them.
static CUtensorMap piece_tmap(const void* ptr, int rows, int H, int hd, long long ld) {
  const uint64_t dims[4] = {static_cast<uint64_t>(hd), static_cast<uint64_t>(H), static_cast<uint64_t>(rows), 1};
  const uint64_t strides[3] = {static_cast<uint64_t>(hd) * 2, static_cast<uint64_t>(ld) * 2, static_cast<uint64_t>(ld) * 2 * static_cast<uint64_t>(rows)};
  const uint32_t box[4] = {64, 1, 32, 1};
  return make_tmap(ptr, 4, dims, strides, box, 2, true);
}

template <int NH>
static void launch_fwd(const PackedAttnArgs& a, cudaStream_t s) {
  constexpr size_t SMEM = 1024 + 2 * NH * HALF_BYTES + FWD_SLOTS * NH * KV_HALF + 8 * NH * 4096 + sizeof(FwdBars);
  static_assert(SMEM <= 232448, "shared memory budget of one CTA exceeded");
  static std::atomic<uint64_t> done{0};
  allow_smem(packed_fwd_kernel<NH>, SMEM, done);
  PackedDev p = make_dev(a);
  p.pair_heads = a.Hq / a.Hkv % 2 == 0 ? 1 : 0;
  p.tiles = p.pair_heads ? a.by_keys : a.pairs;
  p.n_items = p.pair_heads ? a.n_tiles * (a.Hq / 2) : a.n_pairs * a.Hq;
  const CUtensorMap tq = head_tmap(a.q, 1, a.rows, a.Hq, a.hd, a.ld_q), tk = head_tmap(a.k, 1, a.rows, a.Hkv, a.hd, a.ld_k, BKV),
                    tv = head_tmap(a.v, 1, a.rows, a.Hkv, a.hd, a.ld_v, BKV), to = piece_tmap(a.o, a.rows, a.Hq, a.hd, a.ld_o);
  const int grid = p.n_items < num_sms() ? p.n_items : num_sms();
  packed_fwd_kernel<NH><<<grid, FWD_THREADS, SMEM, s>>>(tq, tk, tv, to, p);
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
  static std::atomic<uint64_t> done_kv{0}, done_q{0};
  allow_smem(packed_dkv_kernel<NH>, SMEM_KV, done_kv);
  allow_smem(packed_dq_kernel<NH>, SMEM_Q, done_q);
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
