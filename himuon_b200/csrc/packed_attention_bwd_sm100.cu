// Packed attention, backward pass (formulas, tiles and what is cleared where: packed_attention_sm100.cu).  Two kernels, one block per SM each,
// over lists of items by falling work:
//
// dQ, and delta on the way: an item is a tile of 128 queries of one head; K and V stream through in sub-blocks of 64 positions,
//     S = Q K^T,  dP = dO V^T,   dS = P (dP - delta) written as bf16 over dP's columns in tensor memory,   dQ += dS K.
// dK and dV: an item is a tile of 128 keys of one KV head; Q and dO of the heads of its group stream through, and the scores
// are computed transposed,
//     S^T = K Q^T,  dP^T = V dO^T   (keys on the lanes),   P^T and dS^T over their columns,   dV += P^T dO,  dK += dS^T Q,
// so that every second product has its A operand in tensor memory and dK and dV of all heads of a group meet in one accumulator.
//
// Scores of sub-block i + 1 are issued ahead of the products that need the softmax of sub-block i; 16 warps share each softmax, 16 of the
// 64 columns a group of four.  The next item's loads and scores run beside an item's epilogue.
// A product of 128 x 64 x 16 with both operands in shared memory takes 48 cycles, bound by its operands, one with A in tensor memory 64
// (N = 128): a sub-block needs 1286 cycles of the dK / dV pass and 1029 of the dQ pass, and shared memory is busy for 1280 and 1152 (the
// operands and 32 KB of new ones).  Measured, heads of 128: 1580 and 1280 cycles a sub-block; one document of 8192 tokens, 32 heads over 8, 853 and
// 715 us (802 and 647 TFLOP/s of products, of which P and dP are computed twice), 24 documents of 341 tokens in the mean, 16 over 8, 93 and 85.
// One block for each item and two sub-blocks' scores in all took 990 and 800, 103 and 105: set-up and epilogue were some 10000
// cycles an item, and the softmax of a sub-block on half of the warps took longer than the products beside it.
#include "packed_attention.cuh"

namespace himuon {

namespace {

constexpr int BQ = 64;                               // positions per streamed sub-block
constexpr uint32_t Q_HALF = BQ * 128;                // one 64-column half of a sub-block: 8 KB
constexpr int BWD_THREADS = 576;                     // warp 0: TMA, warp 1: MMA issue, warps 2-17: softmax
constexpr int KV_STAGES = 3;                         // of (Q, dO, log-sum-exp, delta), dK / dV pass
constexpr int Q_STAGES = 4;                          // of (K, V), dQ pass
constexpr uint32_t STAT_BYTES = 2 * BQ * 4;          // minus log-sum-exp[64] then minus delta[64]
// A packed bf16 tile lies over the fp32 columns that its writers have read themselves, 16 of each group: the first 8 of every 16 columns.
__device__ __forceinline__ uint32_t packed_col(int ks) { return static_cast<uint32_t>(ks * 16); }

template <int N>
struct Ring {
  uint32_t at = 0, parity = 0;
  __device__ __forceinline__ Ring next() const {
    Ring r;
    r.at = at == N - 1 ? 0 : at + 1;
    r.parity = at == N - 1 ? parity ^ 1 : parity;
    return r;
  }
};

__device__ __forceinline__ void bulk_load_1d(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// 64 accumulator columns of a warp's 32 rows, scaled, as bf16 to columns `col`.. of a head: by TMA from a 4 KB buffer where all 32 rows are the
// document's, else row by row.  `rows` of them are.
__device__ __forceinline__ void store_head64(const CUtensorMap* tm, __nv_bfloat16* out, long long ld, uint8_t* buf, uint32_t t_src, float scale, int lane,
                                             int rows, int col, int hd, int head, int row0) {
  const bool whole = rows >= 32;                       // uniform over the warp
  tma_store_wait_read<0>();                            // what was here before has left (whichever lane sent it)
  __syncwarp();
#pragma unroll 1
  for (int c = 0; c < 2; ++c) {
    uint32_t v[32];
    tmem_ld32(t_src + c * 32, v);
    tmem_ld_wait();
    if (whole) {
#pragma unroll
      for (int q = 0; q < 4; ++q) *reinterpret_cast<uint4*>(buf + lane * 128 + (((c * 4 + q) ^ (lane & 7)) << 4)) = head8(v + 8 * q, scale);
    } else if (lane < rows) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (col + c * 32 + q * 8 < hd) *reinterpret_cast<uint4*>(out + lane * ld + head * hd + col + c * 32 + q * 8) = head8(v + 8 * q, scale);
    }
  }
  if (whole) {
    fence_proxy_async_smem();
    __syncwarp();
    const uint32_t e = elect_one();
    if (col < hd) tma_store_4d(tm, buf, col, head, row0, 0, e);
    if (e) tma_store_commit();
  }
}

// ================================================================================================ dK and dV
// Tensor memory: S^T buffers at 0 and 64, dP^T at 128 and 192, dV at 256, dK at 384.
struct DkvBars {
  uint64_t kv_full, kv_empty, qd_full[KV_STAGES], qd_empty[KV_STAGES], s_full[2], p_ready[2], acc_done, acc_free;
  uint32_t tmem_slot;
  int abort_flag;
};
struct DkvItem { int first, len, index, slot, hk, h0, heads, subs; };      // heads h0 .. h0 + heads - 1, `subs` sub-blocks of each
__device__ __forceinline__ DkvItem dkv_item(const PackedDev& p, int i) {
  const int per = p.split_heads ? p.Hq : p.Hkv, G = p.Hq / p.Hkv, order = i / per, y = i - order * per;
  const PackedTile t = p.tiles[order];
  DkvItem it;
  it.first = t.first; it.len = t.len; it.index = t.index; it.slot = t.slot;
  it.hk = p.split_heads ? y / G : y;
  it.h0 = p.split_heads ? y : y * G;
  it.heads = p.split_heads ? 1 : G;
  it.subs = (t.len - t.index * AT + BQ - 1) / BQ;      // query sub-blocks from the diagonal to the end
  return it;
}

template <int NH>
__global__ void __launch_bounds__(BWD_THREADS, 1)
packed_dkv_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const __grid_constant__ CUtensorMap tmDO, const __grid_constant__ CUtensorMap tmDK, const __grid_constant__ CUtensorMap tmDV, PackedDev p) {
  constexpr uint32_t TILE_BYTES = NH * HALF_BYTES, Q_TILE = NH * Q_HALF;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_up_1024(smem_raw);
  uint8_t* sK = smem;
  uint8_t* sV = smem + TILE_BYTES;
  uint8_t* sQ = smem + 2 * TILE_BYTES;
  uint8_t* sDO = sQ + KV_STAGES * Q_TILE;
  uint8_t* sOut = sDO + KV_STAGES * Q_TILE;            // 4 KB for each of the 8 NH warps that store
  float* sStat = reinterpret_cast<float*>(sOut + 8 * NH * 4096);
  DkvBars* bars = reinterpret_cast<DkvBars*>(reinterpret_cast<uint8_t*>(sStat) + KV_STAGES * STAT_BYTES);
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = warp_id(), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(&bars->kv_full, 1); mbar_init(&bars->kv_empty, 1);
    for (int i = 0; i < KV_STAGES; ++i) { mbar_init(&bars->qd_full[i], 1); mbar_init(&bars->qd_empty[i], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&bars->s_full[i], 1); mbar_init(&bars->p_ready[i], 512); }
    mbar_init(&bars->acc_done, 1); mbar_init(&bars->acc_free, 512);
    bars->abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) tmem_alloc(&bars->tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, bars->tmem_slot, 0);
  const uint32_t tS = tmem, tDP = tmem + 128, tDV = tmem + 256, tDK = tmem + 384;

  if (warp == 0) {
    // ------------------------------------------------------------ TMA
    const uint32_t e = elect_one();
    Ring<KV_STAGES> r;
    bool ok = true;
    for (int round = 0, i; ok && (i = my_turn(round)) < p.n_items; ++round) {
      const DkvItem it = dkv_item(p, i);
      auto load_stage = [&](int g, int s) {
        if (!mbar_wait_warp(&bars->qd_empty[r.at], r.parity ^ 1, abort_flag, p.status, 4)) return false;
        const int h = it.h0 + g, q0 = it.index * AT + s * BQ;
        uint64_t* bar = &bars->qd_full[r.at];
        mbar_expect_tx(bar, 2 * Q_TILE + STAT_BYTES, e);
        load_head_tile<NH>(sQ + r.at * Q_TILE, Q_HALF, &tmQ, bar, h, it.first + q0, 0, e);
        load_head_tile<NH>(sDO + r.at * Q_TILE, Q_HALF, &tmDO, bar, h, it.first + q0, 0, e);
        const long long stat_idx = h * p.stat_rows + static_cast<long long>(it.slot) * AT + s * BQ;
        if (e) bulk_load_1d(sStat + r.at * 2 * BQ, p.nlse + stat_idx, BQ * 4, bar);
        if (e) bulk_load_1d(sStat + r.at * 2 * BQ + BQ, p.ndelta + stat_idx, BQ * 4, bar);
        r = r.next();
        return true;
      };
      ok = load_stage(0, 0);                           // (ahead of K and V, which wait for the item before)
      if (ok) ok = mbar_wait_warp(&bars->kv_empty, (round & 1) ^ 1, abort_flag, p.status, 4);
      if (!ok) break;
      mbar_expect_tx(&bars->kv_full, 2 * TILE_BYTES, e);
      load_head_tile<NH>(sK, HALF_BYTES, &tmK, &bars->kv_full, it.hk, it.first + it.index * AT, 0, e);
      load_head_tile<NH>(sV, HALF_BYTES, &tmV, &bars->kv_full, it.hk, it.first + it.index * AT, 0, e);
      for (int g = 0; ok && g < it.heads; ++g)
        for (int s = g == 0 ? 1 : 0; ok && s < it.subs; ++s) ok = load_stage(g, s);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issue
    const uint32_t e = elect_one();
    constexpr uint32_t idesc_s = umma_idesc_bf16(128, BQ, false, false);
    constexpr uint32_t idesc_acc = umma_idesc_bf16(128, 64 * NH, false, true);
    const uint64_t k_desc = kmajor_desc(sK), v_desc = kmajor_desc(sV), q_desc = kmajor_desc(sQ), do_desc = kmajor_desc(sDO);
    const uint64_t q_mn = mnmajor_desc(sQ, Q_HALF), do_mn = mnmajor_desc(sDO, Q_HALF);
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity, bool there) { ok = ok && (there || mbar_wait_warp(bar, parity, abort_flag, p.status, 4)); };
    Ring<KV_STAGES> ahead, behind;                     // of the next scores, and of the next products with them
    uint32_t g = 0;                                    // steps of all items
    for (int round = 0, i; ok && (i = my_turn(round)) < p.n_items; ++round) {
      const DkvItem it = dkv_item(p, i);
      const int subs = uniform(it.subs), steps = uniform(it.heads) * subs;
      // positions of a head's last sub-block, if some are missing: the sub-block's rows behind them are the next document's
      const int rest = uniform((it.len - it.index * AT) % BQ);
      int sub = 0;                                     // of the next scores
      bool there = false;                              // their operands
      // Scores of the next sub-block into buffer `b`; `p_bar`: what is waited for after them.
      auto scores = [&](uint32_t b, bool last, uint64_t* p_bar, uint32_t p_par) {
        wait(&bars->qd_full[ahead.at], ahead.parity, there);
        if (!ok) return false;
        if (sub == subs - 1 && rest) {
          clear_rows<NH>(sQ + ahead.at * Q_TILE, Q_HALF, rest, BQ, lane);
          clear_rows<NH>(sDO + ahead.at * Q_TILE, Q_HALF, rest, BQ, lane);
        }
        sub = sub == subs - 1 ? 0 : sub + 1;
        tc_fence_after();
        const uint64_t qd = desc_at(q_desc, ahead.at * Q_TILE), dod = desc_at(do_desc, ahead.at * Q_TILE);
        bool p_there = false;
#pragma unroll
        for (int ks = 0; ks < 4 * NH; ++ks)
          umma_ss(tS + b * BQ, desc_at(k_desc, kmajor_off(HALF_BYTES, ks)), desc_at(qd, kmajor_off(Q_HALF, ks)), idesc_s, ks > 0 ? 1u : 0u, e);
#pragma unroll
        for (int ks = 0; ks < 4 * NH; ++ks) {
          if (ks == 4 * NH - 2 && p_bar) p_there = mbar_peek(p_bar, p_par);
          umma_ss(tDP + b * BQ, desc_at(v_desc, kmajor_off(HALF_BYTES, ks)), desc_at(dod, kmajor_off(Q_HALF, ks)), idesc_s, ks > 0 ? 1u : 0u, e);
        }
        umma_commit(&bars->s_full[b], e);
        if (last) umma_commit(&bars->kv_empty, e);
        ahead = ahead.next();
        return p_there;
      };
      wait(&bars->kv_full, round & 1, false);
      scores(g & 1, steps == 1, nullptr, 0);
      auto step = [&](int j, auto inner) {             // `inner`: neither the first nor the last one
        constexpr bool IN = decltype(inner)::value;
        const uint32_t b = g & 1, p_par = (g >> 1) & 1;
        bool p_there = false;
        if (IN || j + 1 < steps) p_there = scores(b ^ 1, j + 2 == steps, &bars->p_ready[b], p_par);
        if (!IN && j == 0) wait(&bars->acc_free, (round & 1) ^ 1, false);
        wait(&bars->p_ready[b], p_par, p_there);
        if (!ok) return;
        tc_fence_after();
        const uint64_t dod = desc_at(do_mn, behind.at * Q_TILE), qd = desc_at(q_mn, behind.at * Q_TILE);
#pragma unroll
        for (int ks = 0; ks < BQ / 16; ++ks)
          umma_ts(tDV, tS + b * BQ + packed_col(ks), desc_at(dod, mnmajor_off(ks)), idesc_acc, (IN || j > 0 || ks > 0) ? 1u : 0u, e);
        there = false;
#pragma unroll
        for (int ks = 0; ks < BQ / 16; ++ks) {
          if (ks == BQ / 16 - 1) there = (IN || j + 2 < steps) && mbar_peek(&bars->qd_full[ahead.at], ahead.parity);
          umma_ts(tDK, tDP + b * BQ + packed_col(ks), desc_at(qd, mnmajor_off(ks)), idesc_acc, (IN || j > 0 || ks > 0) ? 1u : 0u, e);
        }
        umma_commit(&bars->qd_empty[behind.at], e);
        behind = behind.next();
        ++g;
      };
      int j = 0;
      if (ok) step(j++, std::false_type{});
      for (; ok && j < steps - 1; ++j) step(j, std::true_type{});
      for (; ok && j < steps; ++j) step(j, std::false_type{});
      if (ok) umma_commit(&bars->acc_done, e);
    }
  } else {
    // ------------------------------------------------------------ softmax and epilogue: keys on the lanes
    const int wg = (warp - 2) >> 2, buf = wg & 1, part = wg >> 1;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    if (!p.split_heads) {
      zero_padding(p.dk, p.ld_dk, p.tokens, p.rows, p.Hkv * p.hd, threadIdx.x - 64, 512);
      zero_padding(p.dv, p.ld_dv, p.tokens, p.rows, p.Hkv * p.hd, threadIdx.x - 64, 512);
    }
    const f32x2 scale2 = pack2(p.scale_log2, p.scale_log2);
    bool ok = true;
    uint32_t g0 = 0;                                   // steps of the items before
    Ring<KV_STAGES> r;
    for (int round = 0, i; ok && (i = my_turn(round)) < p.n_items; ++round) {
      const DkvItem it = dkv_item(p, i);
      const int steps = it.heads * it.subs, kv_idx = it.index * AT + row;
      int s = 0;                                       // sub-block of step j
      for (int j = 0; j < steps; ++j, s = s == it.subs - 1 ? 0 : s + 1, r = r.next()) {
        const uint32_t g = g0 + j, b = g & 1, col = b * BQ + wg * 16 + lane_off;
        if (!mbar_wait(&bars->qd_full[r.at], r.parity, abort_flag, p.status, 4)) { ok = false; break; }
        f32x2 nl[8], nd[8];                                     // minus log-sum-exp and minus delta of the columns' queries
        const float* stat = sStat + r.at * 2 * BQ + wg * 16;
#pragma unroll
        for (int t = 0; t < 8; t += 2) {
          const float4 l4 = *reinterpret_cast<const float4*>(stat + 2 * t), d4 = *reinterpret_cast<const float4*>(stat + BQ + 2 * t);
          nl[t] = pack2(l4.x, l4.y); nl[t + 1] = pack2(l4.z, l4.w);
          nd[t] = pack2(d4.x, d4.y); nd[t + 1] = pack2(d4.z, d4.w);
        }
        if (!mbar_wait(&bars->s_full[b], (g >> 1) & 1, abort_flag, p.status, 4)) { ok = false; break; }
        tc_fence_after();
        const int q0 = it.index * AT + s * BQ + wg * 16;
        uint32_t sv[16], dv[16], pk[8], dk[8];
        tmem_ld16(tS + col, sv);
        tmem_ld16(tDP + col, dv);
        tmem_ld_wait();
        float pv[16], ds[16];
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          float x0, x1;
          unpack2(fma2(pack2(sv[2 * t], sv[2 * t + 1]), scale2, nl[t]), x0, x1);
          pv[2 * t] = exp2f(x0);
          pv[2 * t + 1] = exp2f(x1);
          // the softmax scale is applied to dK once, at the end
          unpack2(mul2(pack2(pv[2 * t], pv[2 * t + 1]), add2(nd[t], pack2(dv[2 * t], dv[2 * t + 1]))), ds[2 * t], ds[2 * t + 1]);
        }
        if (s < AT / BQ || q0 + 16 > it.len) {                  // some keys lie after some of these queries, or some queries past the end
#pragma unroll
          for (int t = 0; t < 16; ++t)
            if (q0 + t < kv_idx || q0 + t >= it.len) pv[t] = ds[t] = 0.f;
        }
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          pk[t] = pack_bf16x2(pv[2 * t], pv[2 * t + 1]);
          dk[t] = pack_bf16x2(ds[2 * t], ds[2 * t + 1]);
        }
        tmem_st8(tS + col, pk);                                 // over columns that this thread has read (packed_col)
        tmem_st8(tDP + col, dk);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&bars->p_ready[b]);
      }
      if (!ok || !mbar_wait(&bars->acc_done, round & 1, abort_flag, p.status, 4)) { ok = false; break; }
      tc_fence_after();
      // groups 0 and 2 store dV, 1 and 3 dK, 64 of the columns each
      const int row0 = it.index * AT + (warp & 3) * 32;
      const uint32_t t_src = (buf == 0 ? tDV : tDK) + lane_off + part * 64;
      const float out_scale = buf == 0 ? 1.f : p.scale;
      if (p.split_heads) {
        // this head's part, in 32 bits, (head, row of a tile, column); all heads' meet in sum_heads_kernel
        float* dst = (buf == 0 ? p.dv_part : p.dk_part) + ((it.h0 * p.stat_rows + static_cast<long long>(it.slot) * AT) + row) * p.hd + part * 64;
#pragma unroll 1
        for (int c = 0; c < 64 && part < NH; c += 32) {
          uint32_t v[32];
          tmem_ld32(t_src + c, v);
          tmem_ld_wait();
#pragma unroll
          for (int q = 0; q < 32; q += 4)
            if (part * 64 + c + q < p.hd)
              *reinterpret_cast<float4*>(dst + c + q) = make_float4(__uint_as_float(v[q]) * out_scale, __uint_as_float(v[q + 1]) * out_scale,
                                                                    __uint_as_float(v[q + 2]) * out_scale, __uint_as_float(v[q + 3]) * out_scale);
        }
      } else if (part < NH) {
        const long long ld = buf == 0 ? p.ld_dv : p.ld_dk;
        __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(buf == 0 ? p.dv : p.dk) + static_cast<long long>(it.first + row0) * ld;
        store_head64(buf == 0 ? &tmDV : &tmDK, out, ld, sOut + ((buf * NH + part) * 4 + (warp & 3)) * 4096, t_src, out_scale, lane, it.len - row0, part * 64, p.hd,
                     it.hk, it.first + row0);
      }
      tc_fence_before();
      mbar_arrive(&bars->acc_free);
      g0 += steps;
    }
    tma_store_wait_all();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// dK and dV of a KV head: the sums over its query heads' parts, in their order, four columns a thread.  gridDim.y blocks per tile.
__global__ void __launch_bounds__(256)
sum_heads_kernel(PackedDev p) {
  const PackedTile t = p.tiles[blockIdx.x];
  const int G = p.Hq / p.Hkv, row0 = t.index * AT, rows = min(AT, t.len - row0), per = p.hd / 4;
  const long long stride = p.stat_rows * p.hd;         // from head to head
  for (int i = blockIdx.y * 256 + threadIdx.x; i < rows * p.Hkv * per; i += gridDim.y * 256) {
    const int r = i / (p.Hkv * per), y = i - r * (p.Hkv * per), hk = y / per, c = (y - hk * per) * 4;
    const long long src = hk * G * stride + (static_cast<long long>(t.slot) * AT + r) * p.hd + c, at = t.first + row0 + r;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const float* part = which ? p.dk_part : p.dv_part;
      float4 a = *reinterpret_cast<const float4*>(part + src);
      for (int g = 1; g < G; ++g) {
        const float4 b = *reinterpret_cast<const float4*>(part + src + g * stride);
        a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
      }
      __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(which ? p.dk : p.dv) + at * (which ? p.ld_dk : p.ld_dv) + hk * p.hd + c;
      *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w));
    }
  }
  if (blockIdx.y == 0) {
    zero_padding(p.dk, p.ld_dk, p.tokens, p.rows, p.Hkv * p.hd, threadIdx.x, 256);
    zero_padding(p.dv, p.ld_dv, p.tokens, p.rows, p.Hkv * p.hd, threadIdx.x, 256);
  }
}

// ================================================================================================ dQ
// Tensor memory: three buffers of S and dP, 64 columns each, at 0, 128 and 256, dQ at 384.  Scores run two sub-blocks ahead, so that a softmax
// has a sub-block's time to spare.  Eight more warps compute delta, an item ahead, and store dQ, an item behind.
constexpr int DQ_THREADS = BWD_THREADS + 256;
constexpr int Q_BUFS = 3;
struct DqBars {
  uint64_t qd_full, qd_empty, kv_full[Q_STAGES], kv_empty[Q_STAGES], s_full[Q_BUFS], p_ready[Q_BUFS], acc_done, acc_free, delta_ready[2];
  uint32_t tmem_slot;
  int abort_flag;
  float ndelta[2][AT];                                 // minus delta, of even and odd items
};
struct DqItem { int first, len, index, slot, head, hk, n; };      // n: key sub-blocks up to and including the diagonal
__device__ __forceinline__ DqItem dq_item(const PackedDev& p, int i) {
  const int order = i / p.Hq;
  const PackedTile t = p.tiles[order];
  DqItem it;
  it.first = t.first; it.len = t.len; it.index = t.index; it.slot = t.slot;
  it.head = i - order * p.Hq;
  it.hk = it.head / (p.Hq / p.Hkv);
  it.n = min((t.index + 1) * (AT / BQ), (t.len + BQ - 1) / BQ);
  return it;
}

template <int NH>
__global__ void __launch_bounds__(DQ_THREADS, 1)
packed_dq_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                 const __grid_constant__ CUtensorMap tmDO, const __grid_constant__ CUtensorMap tmDQ, PackedDev p) {
  constexpr uint32_t TILE_BYTES = NH * HALF_BYTES, Q_TILE = NH * Q_HALF;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_up_1024(smem_raw);
  uint8_t* sQ = smem;
  uint8_t* sDO = smem + TILE_BYTES;
  uint8_t* sK = smem + 2 * TILE_BYTES;
  uint8_t* sV = sK + Q_STAGES * Q_TILE;
  uint8_t* sOut = sV + Q_STAGES * Q_TILE;              // 4 KB for each of the 4 NH warps that store
  DqBars* bars = reinterpret_cast<DqBars*>(sOut + 4 * NH * 4096);
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = warp_id(), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(&bars->qd_full, 1); mbar_init(&bars->qd_empty, 1);
    for (int i = 0; i < Q_STAGES; ++i) { mbar_init(&bars->kv_full[i], 1); mbar_init(&bars->kv_empty[i], 1); }
    for (int i = 0; i < Q_BUFS; ++i) { mbar_init(&bars->s_full[i], 1); mbar_init(&bars->p_ready[i], 512); }
    mbar_init(&bars->acc_done, 1); mbar_init(&bars->acc_free, 256);
    for (int i = 0; i < 2; ++i) mbar_init(&bars->delta_ready[i], 256);
    bars->abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) tmem_alloc(&bars->tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, bars->tmem_slot, 0);
  const uint32_t tDQ = tmem + 384;                     // S of buffer b at b * 128, dP 64 columns behind

  if (warp == 0) {
    // ------------------------------------------------------------ TMA
    const uint32_t e = elect_one();
    Ring<Q_STAGES> r;
    bool ok = true;
    for (int round = 0, i; ok && (i = my_turn(round)) < p.n_items; ++round) {
      const DqItem it = dq_item(p, i);
      auto load_stage = [&](int j) {
        if (!mbar_wait_warp(&bars->kv_empty[r.at], r.parity ^ 1, abort_flag, p.status, 4)) return false;
        uint64_t* bar = &bars->kv_full[r.at];
        mbar_expect_tx(bar, 2 * Q_TILE, e);
        load_head_tile<NH>(sK + r.at * Q_TILE, Q_HALF, &tmK, bar, it.hk, it.first + j * BQ, 0, e);
        load_head_tile<NH>(sV + r.at * Q_TILE, Q_HALF, &tmV, bar, it.hk, it.first + j * BQ, 0, e);
        r = r.next();
        return true;
      };
      ok = load_stage(0);                              // (ahead of Q and dO, which wait for the item before)
      if (ok) ok = mbar_wait_warp(&bars->qd_empty, (round & 1) ^ 1, abort_flag, p.status, 4);
      if (!ok) break;
      mbar_expect_tx(&bars->qd_full, 2 * TILE_BYTES, e);
      load_head_tile<NH>(sQ, HALF_BYTES, &tmQ, &bars->qd_full, it.head, it.first + it.index * AT, 0, e);
      load_head_tile<NH>(sDO, HALF_BYTES, &tmDO, &bars->qd_full, it.head, it.first + it.index * AT, 0, e);
      for (int j = 1; ok && j < it.n; ++j) ok = load_stage(j);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issue
    const uint32_t e = elect_one();
    constexpr uint32_t idesc_s = umma_idesc_bf16(128, BQ, false, false);
    constexpr uint32_t idesc_acc = umma_idesc_bf16(128, 64 * NH, false, true);
    const uint64_t q_desc = kmajor_desc(sQ), do_desc = kmajor_desc(sDO), k_desc = kmajor_desc(sK), v_desc = kmajor_desc(sV);
    const uint64_t k_mn = mnmajor_desc(sK, Q_HALF);
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity, bool there) { ok = ok && (there || mbar_wait_warp(bar, parity, abort_flag, p.status, 4)); };
    Ring<Q_STAGES> ahead, behind;                      // operands of the next scores, of the next product with them
    Ring<Q_BUFS> scored, summed;                       // their buffers
    for (int round = 0, i; ok && (i = my_turn(round)) < p.n_items; ++round) {
      const DqItem it = dq_item(p, i);
      const int n = uniform(it.n), rest = uniform(min(it.len - (it.n - 1) * BQ, BQ));      // positions of the last sub-block
      bool there = false;
      // The next scores; `last`: the last ones that need Q and dO.  Returns whether `p_bar`, what is waited for behind them, is there already.
      auto scores = [&](bool last, uint64_t* p_bar, uint32_t p_par) {
        wait(&bars->kv_full[ahead.at], ahead.parity, there);
        if (!ok) return false;
        if (last && rest < BQ) clear_rows<NH>(sK + ahead.at * Q_TILE, Q_HALF, rest, BQ, lane);
        tc_fence_after();
        const uint64_t kd = desc_at(k_desc, ahead.at * Q_TILE), vd = desc_at(v_desc, ahead.at * Q_TILE);
        const uint32_t tS = tmem + scored.at * 128;
        bool p_there = false;
#pragma unroll
        for (int ks = 0; ks < 4 * NH; ++ks)
          umma_ss(tS, desc_at(q_desc, kmajor_off(HALF_BYTES, ks)), desc_at(kd, kmajor_off(Q_HALF, ks)), idesc_s, ks > 0 ? 1u : 0u, e);
#pragma unroll
        for (int ks = 0; ks < 4 * NH; ++ks) {
          if (ks == 4 * NH - 2 && p_bar) p_there = mbar_peek(p_bar, p_par);
          umma_ss(tS + 64, desc_at(do_desc, kmajor_off(HALF_BYTES, ks)), desc_at(vd, kmajor_off(Q_HALF, ks)), idesc_s, ks > 0 ? 1u : 0u, e);
        }
        umma_commit(&bars->s_full[scored.at], e);
        if (last) umma_commit(&bars->qd_empty, e);
        ahead = ahead.next();
        scored = scored.next();
        return p_there;
      };
      wait(&bars->qd_full, round & 1, false);
      scores(n == 1, nullptr, 0);
      if (n > 1) scores(n == 2, nullptr, 0);
      auto step = [&](int j, auto inner) {             // `inner`: neither the first nor one of the last two
        constexpr bool IN = decltype(inner)::value;
        uint64_t* p_bar = &bars->p_ready[summed.at];
        bool p_there = false;
        if (IN || j + 2 < n) p_there = scores(j + 3 == n, p_bar, summed.parity);
        if (!IN && j == 0) wait(&bars->acc_free, (round & 1) ^ 1, false);
        wait(p_bar, summed.parity, p_there);
        if (!ok) return;
        tc_fence_after();
        const uint64_t kd = desc_at(k_mn, behind.at * Q_TILE);
        const uint32_t tDS = tmem + summed.at * 128 + 64;
        there = false;
#pragma unroll
        for (int ks = 0; ks < BQ / 16; ++ks) {
          if (ks == BQ / 16 - 1) there = (IN || j + 3 < n) && mbar_peek(&bars->kv_full[ahead.at], ahead.parity);
          umma_ts(tDQ, tDS + packed_col(ks), desc_at(kd, mnmajor_off(ks)), idesc_acc, (IN || j > 0 || ks > 0) ? 1u : 0u, e);
        }
        umma_commit(&bars->kv_empty[behind.at], e);
        behind = behind.next();
        summed = summed.next();
      };
      int j = 0;
      if (ok) step(j++, std::false_type{});
      for (; ok && j < n - 2; ++j) step(j, std::true_type{});
      for (; ok && j < n; ++j) step(j, std::false_type{});
      if (ok) umma_commit(&bars->acc_done, e);
    }
  } else if (warp < 18) {
    // ------------------------------------------------------------ softmax: queries on the lanes
    const int wg = (warp - 2) >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    zero_padding(p.dq, p.ld_dq, p.tokens, p.rows, p.Hq * p.hd, threadIdx.x - 64, 512);
    const f32x2 scale2 = pack2(p.scale_log2, p.scale_log2);
    auto row_stat = [&](const DqItem& it) { return p.nlse[it.head * p.stat_rows + static_cast<long long>(it.slot) * AT + row]; };
    bool ok = true;
    Ring<Q_BUFS> r;
    int i = my_turn(0);
    DqItem it{};
    float nlse = 0.f;
    if (i < p.n_items) {
      it = dq_item(p, i);
      nlse = row_stat(it);
    }
    for (int round = 0; ok && i < p.n_items; ++round) {
      const int n = it.n, first_masked = it.index * AT, q_idx = it.index * AT + row;
      const f32x2 nlse_2 = pack2(nlse, nlse);
      i = my_turn(round + 1);                          // what the next item needs from memory is fetched while this one runs
      if (i < p.n_items) {
        it = dq_item(p, i);
        nlse = row_stat(it);
      }
      if (!mbar_wait(&bars->delta_ready[round & 1], (round >> 1) & 1, abort_flag, p.status, 4)) break;
      const float ndelta = bars->ndelta[round & 1][row];
      const f32x2 ndelta_2 = pack2(ndelta, ndelta);
      for (int j = 0; j < n; ++j, r = r.next()) {
        const uint32_t tS = tmem + r.at * 128 + wg * 16 + lane_off;
        if (!mbar_wait(&bars->s_full[r.at], r.parity, abort_flag, p.status, 4)) { ok = false; break; }
        tc_fence_after();
        const int kv0 = j * BQ + wg * 16;
        uint32_t sv[16], dv[16], dk[8];
        tmem_ld16(tS, sv);
        tmem_ld16(tS + 64, dv);
        tmem_ld_wait();
        float ds[16];
#pragma unroll
        for (int t = 0; t < 16; t += 2) {
          float x0, x1;
          unpack2(fma2(pack2(sv[t], sv[t + 1]), scale2, nlse_2), x0, x1);
          unpack2(mul2(pack2(exp2f(x0), exp2f(x1)), add2(pack2(dv[t], dv[t + 1]), ndelta_2)), ds[t], ds[t + 1]);
        }
        if (kv0 + 15 > first_masked) {                          // some of these keys lie after some queries
#pragma unroll
          for (int t = 0; t < 16; ++t)
            if (kv0 + t > q_idx) ds[t] = 0.f;
        }
#pragma unroll
        for (int t = 0; t < 8; ++t) dk[t] = pack_bf16x2(ds[2 * t], ds[2 * t + 1]);
        tmem_st8(tS + 64, dk);                                  // over columns that this thread has read (packed_col)
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&bars->p_ready[r.at]);
      }
    }
  } else {
    // ------------------------------------------------------------ delta ahead, dQ behind
    constexpr int LPR = 8 * NH, RPP = 32 / LPR;        // lanes per row, rows per pass
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const int part = (warp - 18) >> 2;                 // two warps for the same 32 lanes: 16 rows of delta, 64 columns of dQ each
    uint8_t* stage = sOut + (part * 4 + (warp & 3)) * 4096;
    // delta = sum over the head of O dO, 8 columns a lane; O with the bits that its bf16 lacks (low_of)
    auto delta_of = [&](const DqItem& it, int round) {
      constexpr int BATCH = 4;                         // passes whose loads are on their way together
      const int c = (lane % LPR) * 8, r0 = (warp & 3) * 32 + part * 16 + lane / LPR;
      const __nv_bfloat16* o = reinterpret_cast<const __nv_bfloat16*>(p.o_in) + it.head * p.hd + c;
      const __nv_bfloat16* g = reinterpret_cast<const __nv_bfloat16*>(p.d_o) + it.head * p.hd + c;
#pragma unroll 1
      for (int k0 = 0; k0 < 16; k0 += BATCH * RPP) {
        uint4 o4[BATCH], g4[BATCH];
        uint2 l2[BATCH];
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
          const int at = it.index * AT + r0 + k0 + k * RPP;
          o4[k] = g4[k] = make_uint4(0, 0, 0, 0);
          l2[k] = make_uint2(0, 0);
          if (at < it.len && c < p.hd) {
            o4[k] = *reinterpret_cast<const uint4*>(o + static_cast<long long>(it.first + at) * p.ld_o);
            g4[k] = *reinterpret_cast<const uint4*>(g + static_cast<long long>(it.first + at) * p.ld_do);
            l2[k] = *reinterpret_cast<const uint2*>(p.o_low + low_at(p, it.head, it.slot, r0 + k0 + k * RPP, c));
          }
        }
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
          const uint32_t ow[4] = {o4[k].x, o4[k].y, o4[k].z, o4[k].w}, gw[4] = {g4[k].x, g4[k].y, g4[k].z, g4[k].w};
          float d = 0.f;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint32_t low = q < 2 ? l2[k].x : l2[k].y, lo = ow[q] << 16, hi = ow[q] & 0xFFFF0000u;
            d += (q & 1 ? with_low<2>(lo, low) : with_low<0>(lo, low)) * bf16_lo(gw[q]) + (q & 1 ? with_low<3>(hi, low) : with_low<1>(hi, low)) * bf16_hi(gw[q]);
          }
#pragma unroll
          for (int x = LPR / 2; x > 0; x >>= 1) d += __shfl_xor_sync(0xffffffffu, d, x);
          if (lane % LPR == 0) {
            bars->ndelta[round & 1][r0 + k0 + k * RPP] = -d;
            p.ndelta[it.head * p.stat_rows + static_cast<long long>(it.slot) * AT + r0 + k0 + k * RPP] = -d;
          }
        }
      }
      mbar_arrive(&bars->delta_ready[round & 1]);
    };
    int i = my_turn(0);
    DqItem it{};
    if (i < p.n_items) {
      it = dq_item(p, i);
      delta_of(it, 0);
    }
    for (int round = 0; i < p.n_items; ++round) {
      const DqItem now = it;
      i = my_turn(round + 1);
      if (i < p.n_items) {
        it = dq_item(p, i);
        delta_of(it, round + 1);                       // (its place was the item before last's, whose dQ has been stored)
      }
      if (!mbar_wait(&bars->acc_done, round & 1, abort_flag, p.status, 4)) break;
      tc_fence_after();
      const int row0 = now.index * AT + (warp & 3) * 32;
      // dS was left unscaled, so the softmax scale lands here
      if (part < NH)
        store_head64(&tmDQ, reinterpret_cast<__nv_bfloat16*>(p.dq) + static_cast<long long>(now.first + row0) * p.ld_dq, p.ld_dq, stage,
                     tDQ + part * 64 + lane_off, p.scale, lane, now.len - row0, part * 64, p.hd, now.head, now.first + row0);
      tc_fence_before();
      mbar_arrive(&bars->acc_free);
    }
    tma_store_wait_all();
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
template <int NH>
static void launch_bwd(const PackedAttnArgs& a, cudaStream_t s) {
  constexpr size_t SMEM_KV = 1024 + 2 * NH * HALF_BYTES + 2 * KV_STAGES * NH * Q_HALF + 8 * NH * 4096 + KV_STAGES * STAT_BYTES + sizeof(DkvBars);
  constexpr size_t SMEM_Q = 1024 + 2 * NH * HALF_BYTES + 2 * Q_STAGES * NH * Q_HALF + 4 * NH * 4096 + sizeof(DqBars);
  static_assert(SMEM_KV <= 232448 && SMEM_Q <= 232448, "shared memory budget of one CTA exceeded");
  static std::atomic<uint64_t> done_kv{0}, done_q{0};
  allow_smem(packed_dkv_kernel<NH>, SMEM_KV, done_kv);
  allow_smem(packed_dq_kernel<NH>, SMEM_Q, done_q);
  PackedDev p = make_dev(a);
  const CUtensorMap tq = head_tmap(a.q, 1, a.rows, a.Hq, a.hd, a.ld_q), tdo = head_tmap(a.d_o, 1, a.rows, a.Hq, a.hd, a.ld_do),
                    tk = head_tmap(a.k, 1, a.rows, a.Hkv, a.hd, a.ld_k), tv = head_tmap(a.v, 1, a.rows, a.Hkv, a.hd, a.ld_v),
                    tq64 = head_tmap(a.q, 1, a.rows, a.Hq, a.hd, a.ld_q, BQ), tdo64 = head_tmap(a.d_o, 1, a.rows, a.Hq, a.hd, a.ld_do, BQ),
                    tk64 = head_tmap(a.k, 1, a.rows, a.Hkv, a.hd, a.ld_k, BQ), tv64 = head_tmap(a.v, 1, a.rows, a.Hkv, a.hd, a.ld_v, BQ),
                    tdq = head_tmap(a.dq, 1, a.rows, a.Hq, a.hd, a.ld_dq, 32), tdk = head_tmap(a.dk, 1, a.rows, a.Hkv, a.hd, a.ld_dk, 32),
                    tdv = head_tmap(a.dv, 1, a.rows, a.Hkv, a.hd, a.ld_dv, 32);
  auto grid = [&] { return p.n_items < num_sms() ? p.n_items : num_sms(); };
  p.tiles = a.by_keys;
  p.n_items = a.n_tiles * a.Hq;
  packed_dq_kernel<NH><<<grid(), DQ_THREADS, SMEM_Q, s>>>(tq, tk64, tv64, tdo, tdq, p);      // and delta, which the other reads
  check_packed_launch("dQ");
  p.tiles = a.by_queries;
  p.split_heads = a.dkv_part != nullptr ? 1 : 0;
  p.dk_part = a.dkv_part;
  p.dv_part = a.dkv_part ? a.dkv_part + p.stat_rows * a.Hq * a.hd : nullptr;
  p.n_items = a.n_tiles * (p.split_heads ? a.Hq : a.Hkv);
  packed_dkv_kernel<NH><<<grid(), BWD_THREADS, SMEM_KV, s>>>(tq64, tk, tv, tdo64, tdk, tdv, p);
  check_packed_launch("dK / dV");
  if (p.split_heads) {
    sum_heads_kernel<<<dim3(a.n_tiles, (AT * a.Hkv * (a.hd / 4) + 255) / 256), 256, 0, s>>>(p);
    check_packed_launch("sum over heads");
  }
}
void packed_attn_bwd(const PackedAttnArgs& a, cudaStream_t s) {
  check_packed(a);
  if (a.n_tiles == 0) return;
  if (head_halves(a.hd) == 1) launch_bwd<1>(a, s);
  else launch_bwd<2>(a, s);
}

}  // namespace himuon
