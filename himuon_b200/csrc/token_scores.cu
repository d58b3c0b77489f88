// Log probability of given tokens, entropy and likeliest alternatives of rows of logits (bf16 or fp32), and the gradient
// that reaches the logits.
//
// With m = max x, d = x - m:   s = sum e^d,  t = sum d e^d,   log p_j = d_j - log s,   H = log s - t / s.
// Shifted by the maximum both sums have terms of one sign, so the entropy of a peaked row loses nothing to cancellation, and
// partial results merge: moving (m1, s1, t1) to a larger m scales s1 by f = e^(m1-m) and turns t1 into f (t1 + (m1-m) s1).
// Gradient, with the incoming g of log p_y and h of H:   dx_j = g [j = y] - p_j (g + h (log p_j + H)).  (token_scores.cuh)
// A logit of -inf has p = 0 and no part in H.  A row of nothing but -inf has log p = -inf, H = 0 and no gradient.  An id equal to
// `ignore` has log p = 0 and passes no g on; an id outside the vocabulary has log p = NaN and passes none on either.
//
// One pass over the logits.  fp32 logits run at the rate of memory (2048 x 151936: 178 us, 7.0 TB/s); bf16 ones come close to what the
// SMs can exponentiate, 16 a clock (2048 x 151936: 105 to 116 us, 5.4 to 5.9 TB/s, exponential unit 63 to 72 % busy), and alternatives cost half as much
// again (1024 x 128256 with 8: 66 us, where 46 would do without; of that a third at a row's start and end).  A row goes to a cluster of 1 to 8 blocks, so that a few
// rows occupy the GPU as well (scores_split()); the blocks' partial results meet in distributed shared memory.  The gradient, one read
// and one write, takes 215 us at 2048 x 151936 bf16 (5.8 TB/s).
// Likeliest alternatives: each warp keeps a sorted list of 32, one a lane, as 64-bit keys of value and inverted index, so that equal
// values go to the lower index.  What passes a floor that all warps raise together is collected in shared memory and merged 32 at a
// time by a bitonic network.
#include <stdint.h>

#include "himuon.h"
#include "pair_common.cuh"
#include "sm100_common.cuh"
#include "token_scores.cuh"

namespace himuon {

namespace {

constexpr int NW = 8, NT = NW * 32;              // warps and threads of a block
template <typename T> struct Vec;                 // one 16-byte group of logits
template <> struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[4]) {
    f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ float one(const float* p) { return *p; }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[8]) {
    f[0] = bf16_lo(u.x); f[1] = bf16_hi(u.x); f[2] = bf16_lo(u.y); f[3] = bf16_hi(u.y);
    f[4] = bf16_lo(u.z); f[5] = bf16_hi(u.z); f[6] = bf16_lo(u.w); f[7] = bf16_hi(u.w);
  }
  static __device__ __forceinline__ float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
};

// ---------------------------------------------------------------- lists of the largest
typedef unsigned long long Key;
__device__ __forceinline__ Key key_of(float x, uint32_t index) {
  uint32_t b = __float_as_uint(x);
  if ((b << 1) == 0) b = 0;                                          // -0 is 0
  if ((b << 1) > 0xFF000000u) b = 0x7FFFFFFFu;                       // NaN is above everything
  b = (b >> 31) ? ~b : (b | 0x80000000u);
  return (static_cast<Key>(b) << 32) | ~index;
}
__device__ __forceinline__ float key_value(Key k) {
  const uint32_t b = static_cast<uint32_t>(k >> 32);
  return __uint_as_float((b >> 31) ? (b & 0x7FFFFFFFu) : ~b);
}
__device__ __forceinline__ uint32_t key_index(Key k) { return ~static_cast<uint32_t>(k); }

// `k` over the lanes, a bitonic sequence, into descending order.
__device__ __forceinline__ Key bitonic_down(Key k, int lane) {
#pragma unroll
  for (int j = 16; j > 0; j >>= 1) {
    const Key o = __shfl_xor_sync(0xffffffffu, k, j);
    k = ((lane & j) == 0) == (k > o) ? k : o;
  }
  return k;
}
__device__ __forceinline__ Key sorted_down(Key k, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1) {
#pragma unroll
    for (int j = size >> 1; j > 0; j >>= 1) {
      const Key o = __shfl_xor_sync(0xffffffffu, k, j);
      const bool down = (lane & size) == 0 || size == 32;
      k = (((lane & j) == 0) == down) == (k > o) ? k : o;
    }
  }
  return k;
}
// The 32 largest of two descending lists, descending.
__device__ __forceinline__ Key merged_down(Key a, Key b, int lane) {
  const Key r = __shfl_sync(0xffffffffu, b, 31 - lane);
  return bitonic_down(a > r ? a : r, lane);
}

struct TopList {
  Key best;              // this lane's entry
  Key kth;               // the k-th of the list
  int waiting;           // entries of `buf` in use, the same in all lanes
  Key* buf;              // 64 of this warp
  int lane, k;
  __device__ __forceinline__ void start(Key* b, int l, int k_) {
    best = 0; kth = 0; waiting = 0; buf = b; lane = l; k = k_;
  }
  __device__ __forceinline__ void flush() {
    __syncwarp();
    const Key x = lane < waiting ? buf[lane] : 0;
    const Key rest = lane + 32 < waiting ? buf[lane + 32] : 0;
    __syncwarp();
    buf[lane] = rest;
    __syncwarp();                // (the exchanges below order no memory, and the next push of another lane may go to this slot)
    best = merged_down(best, sorted_down(x, lane), lane);
    kth = __shfl_sync(0xffffffffu, best, k - 1);
    waiting = waiting > 32 ? waiting - 32 : 0;
  }
  // One key a lane, 0 for none; called by the whole warp.
  __device__ __forceinline__ void push(Key key) {
    const bool in = key > kth;
    const uint32_t who = __ballot_sync(0xffffffffu, in);
    if (in) buf[waiting + __popc(who & ((1u << lane) - 1))] = key;
    waiting += __popc(who);
    if (waiting > 32) flush();
  }
};

// A float in an order that unsigned words have, and a word a lane into descending order.
__device__ __forceinline__ uint32_t word_of(float x) { return static_cast<uint32_t>(key_of(x, 0) >> 32); }
__device__ __forceinline__ uint32_t sorted_down(uint32_t k, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1) {
#pragma unroll
    for (int j = size >> 1; j > 0; j >>= 1) {
      const uint32_t o = __shfl_xor_sync(0xffffffffu, k, j);
      k = (((lane & j) == 0) == ((lane & size) == 0 || size == 32)) ? max(k, o) : min(k, o);
    }
  }
  return k;
}

// The largest over the lanes, taken away from the first lane that has it.
__device__ __forceinline__ uint32_t take_largest(uint32_t& u, int lane) {
  const uint32_t top = __reduce_max_sync(0xffffffffu, u), who = __ballot_sync(0xffffffffu, u == top);
  if (lane == __ffs(who) - 1) u = 0;
  return top;
}

}  // namespace

struct ScoreArgsDev {
  const void* logits;
  const long long* ids;
  float* log_probs;
  float* entropy;
  float2* stats;             // (m, log s) of each row, for the gradient
  float* top_log_probs;
  long long* top_ids;
  long long rows, ld, ignore;
  int vocab, k;
};

__device__ __forceinline__ uint32_t cluster_nctas() {
  uint32_t n;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n));
  return n;
}
template <typename V>
__device__ __forceinline__ V load_remote(const V* p, uint32_t rank) {     // a multiple of 4 bytes from another block's shared memory
  V out;
  uint32_t* w = reinterpret_cast<uint32_t*>(&out);
  const uint32_t a = map_to_cta(smem_u32(p), rank);
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(V) / 4); ++i)
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(w[i]) : "r"(a + 4 * i) : "memory");
  return out;
}

// The warps' lists, one entry a lane, merged into warp 0's `best`.
__device__ __forceinline__ void join_lists(Key& best, Key (*lists)[32], int warp, int lane) {
#pragma unroll
  for (int o = NW / 2; o > 0; o >>= 1) {
    __syncthreads();
    if (warp >= o && warp < 2 * o) lists[warp][lane] = best;
    __syncthreads();
    if (warp < o) best = merged_down(best, lists[warp + o][lane], lane);
  }
}

__device__ __forceinline__ void copy_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Cluster = one row.  Block r of the cluster takes the r-th share of the row's whole 16-byte groups; what lies before the first
// group and behind the last goes to the first block.
// With alternatives: a thread's maximum so far is that of an element of its own, so the k-th largest of all warps' four largest thread
// maxima is a value that k elements reach.  Nothing below it can be among the k; the warps publish and read them as they go (they only
// grow, so old ones are still true), and after the first pass over the block's threads few threads have a candidate.
template <typename T, bool TOP>
__global__ void __launch_bounds__(NT, 4)
token_scores_kernel(ScoreArgsDev p) {
  constexpr int N = Vec<T>::N, UN = 4, RING = 2;
  // Up to FEW threads with candidates are looked through one after the other by the whole warp, more than that each through its own: 1024 x 128256
  // with 8 alternatives 65 us (70 the second way always), 512 x 1024 with 5 12 us (17 the first way always).
  // A warp looks the floor up again after RENEW threads with candidates: 1024 x 128256 with 1 / 8 / 20 59 / 66 / 71 us (65 / 65 / 74 by every
  // second pass and the least of the warps' maxima).
  constexpr int FEW = 2, RENEW = 8;
  __shared__ uint4 s_ring[RING][UN][NT];
  __shared__ Sums s_sums[NW];
  __shared__ Sums s_block;
  __shared__ Key s_buf[TOP ? NW * 64 : 1];
  __shared__ Key s_lists[TOP ? NW : 1][32];
  __shared__ volatile uint32_t s_high[NW * 4];      // each warp's four largest thread maxima
  constexpr int POOL = 96;
  __shared__ Key s_pool[TOP ? POOL : 1];
  __shared__ int s_count;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t parts = cluster_nctas(), part = cluster_ctarank();
  const long long row = blockIdx.x / parts;
  const T* x = reinterpret_cast<const T*>(p.logits) + row * p.ld;
  // elements before the first 16-byte boundary (rows of an odd vocabulary start anywhere)
  int head = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / static_cast<int>(sizeof(T));
  if (head > p.vocab) head = p.vocab;
  const int groups = (p.vocab - head) / N;
  const int g0 = static_cast<int>(static_cast<long long>(groups) * part / parts), g1 = static_cast<int>(static_cast<long long>(groups) * (part + 1) / parts);
  const uint4* body = reinterpret_cast<const uint4*>(x + head);

  // the row's own token, fetched while the rest is on its way
  float own = nan_f();
  bool counted = false;
  if (part == 0 && threadIdx.x == 0) {
    const long long y = p.ids[row];
    counted = y != p.ignore;
    if (counted && y >= 0 && y < p.vocab) own = Vec<T>::one(x + y);
  }
  Sums a{-INFINITY, 0.f, 0.f};
  TopList top;
  float floor = -INFINITY;
  int seen = 0;                                     // candidates' threads since the floor was looked up
  if (TOP) {
    top.start(s_buf + warp * 64, lane, p.k);
    if (threadIdx.x == 0) s_count = 0;
    __syncthreads();
  }
  // Each thread copies its own groups to shared memory ahead of their use and is the only one to read them, so that the copies
  // wait for nothing but themselves.  (Loads into registers, one pass in flight and then none:
  // 123 us for 1024 x 128256 with 8 alternatives, 107 this way.)
  auto group_of = [&](int pass, int u) { return g0 + ((pass * NW + warp) * UN + u) * 32 + lane; };
  const int passes = (g1 - g0 + NT * UN - 1) / (NT * UN);        // of the block, the same for every warp
  auto fetch = [&](int pass) {
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int i = group_of(pass, u);
      if (pass < passes && i < g1) copy_async16(&s_ring[pass % RING][u][threadIdx.x], body + i);
    }
    copy_async_commit();
  };
  auto publish = [&] {
    uint32_t rest = word_of(a.m), high = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t most = take_largest(rest, lane);
      high = lane == i ? most : high;
    }
    if (lane < 4) s_high[warp * 4 + lane] = high;
  };
  auto kth_published = [&] {
    uint32_t rest = s_high[lane], kth = 0;
    if (p.k > 12) kth = __shfl_sync(0xffffffffu, sorted_down(rest, lane), p.k - 1);      // (15 exchanges in a row)
    else for (int i = 0; i < p.k; ++i) kth = take_largest(rest, lane);
    return key_value(static_cast<Key>(kth) << 32);
  };
  for (int pass = 0; pass < RING - 1; ++pass) fetch(pass);
  for (int pass = 0; pass < passes; ++pass) {
    fetch(pass + RING - 1);
    copy_async_wait<RING - 1>();
    // all groups of a pass at once: their exponentials do not wait for one another
    float v[UN * N];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      float f[N];
      Vec<T>::unpack(s_ring[pass % RING][u][threadIdx.x], f);
#pragma unroll
      for (int q = 0; q < N; ++q) v[u * N + q] = f[q];
    }
    if (pass == passes - 1) {                         // past the end: whatever the slots hold
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        const bool live = group_of(pass, u) < g1;
#pragma unroll
        for (int q = 0; q < N; ++q) v[u * N + q] = live ? v[u * N + q] : -INFINITY;
      }
    }
    const float most = largest<UN * N>(v);
    take<UN * N>(a, v, most);
    if constexpr (TOP) {
      if (pass == 0 || seen >= RENEW) {
        publish();
        if (pass == 0) __syncthreads();               // the first values of every warp; later ones may be a little old
        else __syncwarp();
        floor = kth_published();
        seen = 0;
      }
      uint32_t who = __ballot_sync(0xffffffffu, most >= floor);
      seen += __popc(who);
      if (__popc(who) > FEW) {                        // every lane goes through its own, one at a time
        uint32_t hits = 0;
#pragma unroll
        for (int q = 0; q < UN * N; ++q) hits |= v[q] >= floor ? 1u << q : 0u;
        if (pass == passes - 1) {
#pragma unroll
          for (int u = 0; u < UN; ++u) if (group_of(pass, u) >= g1) hits &= ~(((1u << N) - 1) << (u * N));
        }
        while (__any_sync(0xffffffffu, hits != 0)) {
          Key key = 0;
          if (hits) {
            const int at = __ffs(hits) - 1, u = at / N, q = at % N;
            hits &= hits - 1;
            const T* slot = reinterpret_cast<const T*>(&s_ring[pass % RING][u][threadIdx.x]);
            key = key_of(Vec<T>::one(slot + q), static_cast<uint32_t>(head + group_of(pass, u) * N + q));
          }
          top.push(key);
        }
      } else if (who) {                               // as a rule: one lane or two, whose logits all lanes look at, one each
        __syncwarp();
        const int u = lane / N % UN, q = lane % N;
        for (; who; who &= who - 1) {
          const int of = __ffs(who) - 1, i = group_of(pass, u) - lane + of;
          const float xq = Vec<T>::one(reinterpret_cast<const T*>(&s_ring[pass % RING][u][warp * 32 + of]) + q);
          top.push(lane < UN * N && i < g1 && xq >= floor ? key_of(xq, static_cast<uint32_t>(head + i * N + q)) : 0);
        }
        __syncwarp();                                 // (the slots are copied to again)
      }
    }
  }
  if (part == 0 && warp == 0) {                     // the ragged ends: fewer than 2 N elements
    const int tail0 = head + groups * N, loose = head + p.vocab - tail0;
    const bool live = lane < loose;
    const int at = lane < head ? lane : tail0 + lane - head;
    float v[2] = {-INFINITY, -INFINITY};
    if (live) v[0] = Vec<T>::one(x + at);
    if (live) take<2>(a, v, v[0]);
    if (TOP) top.push(live ? key_of(v[0], static_cast<uint32_t>(at)) : 0);
  }
  // lanes, warps, blocks
  if (TOP) {
    publish();
  }
  a = lanes_merged(a);
  if (lane == 0) s_sums[warp] = a;
  if constexpr (TOP) {
    // NaN and +inf never raise a floor and are not seen by a comparison with one: such a row (its sum is NaN) is looked through again
    const bool odd = __syncthreads_or(!(a.s >= 0.f));
    if (odd) {
      for (int i0 = g0 + warp * 32; i0 < g1; i0 += NT) {
        const int i = i0 + lane;
        float v[N];
        Vec<T>::unpack(i < g1 ? body[i] : make_uint4(0, 0, 0, 0), v);
        if (i0 == g0 + warp * 32) { top.best = 0; top.kth = 0; top.waiting = 0; }
#pragma unroll 1
        for (int q = 0; q < N; ++q) {
          float xq = v[0];
#pragma unroll
          for (int r = 1; r < N; ++r) xq = r == q ? v[r] : xq;
          top.push(i < g1 ? key_of(xq, static_cast<uint32_t>(head + i * N + q)) : 0);
        }
      }
      if (part == 0 && warp == 0) {
        const int tail0 = head + groups * N, loose = head + p.vocab - tail0;
        const int at = lane < head ? lane : tail0 + lane - head;
        if (g0 + warp * 32 >= g1) { top.best = 0; top.kth = 0; top.waiting = 0; }
        top.push(lane < loose ? key_of(Vec<T>::one(x + at), static_cast<uint32_t>(at)) : 0);
      }
    } else {
      // what reaches the last floor: a few more than k as a rule, few enough for one warp
      floor = kth_published();
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        const Key key = i == 2 ? top.best : lane + 32 * i < top.waiting ? top.buf[lane + 32 * i] : 0;
        if (key != 0 && key_value(key) >= floor) {
          const int at = atomicAdd(&s_count, 1);
          if (at < POOL) s_pool[at] = key;
        }
      }
      __syncthreads();
    }
    const int n = odd ? POOL + 1 : s_count;           // uniform
    if (n <= POOL) {
      if (warp == 0) {
        // (no two keys are alike: each finds its place by itself, without the exchanges in a row of a sort)
        s_lists[0][lane] = 0;
        __syncwarp();
        for (int i = lane; i < n; i += 32) {
          const Key mine = s_pool[i];
          int before = 0;
#pragma unroll 4
          for (int j = 0; j < n; ++j) before += s_pool[j] > mine ? 1 : 0;
          if (before < 32) s_lists[0][before] = mine;
        }
        __syncwarp();
        top.best = s_lists[0][lane];
      }
    } else {
      while (top.waiting > 0) top.flush();
      join_lists(top.best, s_lists, warp, lane);
    }
  }
  __syncthreads();
  if (warp == 0) {
    a = lane < NW ? s_sums[lane] : Sums{-INFINITY, 0.f, 0.f};
    a = lanes_merged(a);
  }
  if (parts > 1) {                                  // uniform over the cluster
    if (warp == 0) {
      if (lane == 0) s_block = a;
      if (TOP) s_lists[0][lane] = top.best;
    }
    cluster_sync_all();
    if (part == 0 && warp == 0) {
      a = static_cast<uint32_t>(lane) < parts ? load_remote(&s_block, lane) : Sums{-INFINITY, 0.f, 0.f};
      a = lanes_merged(a);
    }
    if (TOP && part == 0) top.best = static_cast<uint32_t>(warp) < parts ? load_remote(&s_lists[0][lane], warp) : 0;
    cluster_sync_all();                             // no block leaves while it is still read
    if (TOP && part == 0) join_lists(top.best, s_lists, warp, lane);
  }
  if (part == 0 && warp == 0) {
    const RowScore r = row_score(a);
    if (lane == 0) {
      p.log_probs[row] = counted ? (own - r.m) - r.log_s : 0.f;
      p.entropy[row] = r.entropy;
      if (p.stats) p.stats[row] = make_float2(r.m, r.log_s);
    }
    if (TOP && lane < p.k) {
      p.top_log_probs[row * p.k + lane] = (key_value(top.best) - r.m) - r.log_s;
      p.top_ids[row * p.k + lane] = key_index(top.best);
    }
  }
}

struct ScoreGradDev {
  const void* logits;
  void* grad;
  const long long* ids;
  const float* entropy;
  const float2* stats;
  const float* g_log_probs;     // either may be null
  const float* g_entropy;
  long long rows, ld, ld_grad, ignore;
  int vocab;
};

template <typename D>
__device__ __forceinline__ void store_one(D* p, float v);
template <>
__device__ __forceinline__ void store_one<float>(float* p, float v) { *p = v; }
template <>
__device__ __forceinline__ void store_one<__nv_bfloat16>(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// T: logits, D: gradient.  Rows that share the offset from 16 bytes with the gradient's are read and written in 16-byte groups of
// logits; others element by element.
constexpr int SG_GROUPS = 4;                        // 16-byte groups of logits a thread takes
template <typename T, typename D>
__global__ void __launch_bounds__(NT)
token_scores_grad_kernel(ScoreGradDev p, int blocks_per_row) {
  constexpr int N = Vec<T>::N;
  const long long row = blockIdx.x / blocks_per_row;
  const int piece = static_cast<int>(blockIdx.x - row * blocks_per_row);
  const T* x = reinterpret_cast<const T*>(p.logits) + row * p.ld;
  D* dx = reinterpret_cast<D*>(p.grad) + row * p.ld_grad;
  const RowGrad r = row_grad(p.stats, p.entropy, p.ids, p.g_log_probs, p.g_entropy, p.ignore, p.vocab, row);

  int head = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / static_cast<int>(sizeof(T));
  if (head > p.vocab) head = p.vocab;
  const bool wide = (reinterpret_cast<uintptr_t>(dx + head) & (N * sizeof(D) - 1) & 15) == 0;
  const int groups = (p.vocab - head) / N;
#pragma unroll
  for (int u = 0; u < SG_GROUPS; ++u) {
    const int i = (piece * SG_GROUPS + u) * NT + static_cast<int>(threadIdx.x);
    if (i >= groups) break;
    const int at = head + i * N;
    float v[N], d[N];
    Vec<T>::unpack(__ldcs(reinterpret_cast<const uint4*>(x + head) + i), v);
#pragma unroll
    for (int q = 0; q < N; ++q) d[q] = grad_of(r, v[q], at + q);
    if (wide) {
      if constexpr (sizeof(D) == 4) {
#pragma unroll
        for (int q = 0; q < N; q += 4) *reinterpret_cast<float4*>(dx + at + q) = make_float4(d[q], d[q + 1], d[q + 2], d[q + 3]);
      } else if constexpr (N == 8) {
        *reinterpret_cast<uint4*>(dx + at) = make_uint4(pack_bf16x2(d[0], d[1]), pack_bf16x2(d[2], d[3]), pack_bf16x2(d[4], d[5]), pack_bf16x2(d[6], d[7]));
      } else {
        *reinterpret_cast<uint2*>(dx + at) = make_uint2(pack_bf16x2(d[0], d[1]), pack_bf16x2(d[2], d[3]));
      }
    } else {
#pragma unroll
      for (int q = 0; q < N; ++q) store_one<D>(dx + at + q, d[q]);
    }
  }
  const int tail0 = head + groups * N, loose = head + p.vocab - tail0;
  if (piece == 0 && static_cast<int>(threadIdx.x) < loose) {
    const int at = static_cast<int>(threadIdx.x) < head ? threadIdx.x : tail0 + threadIdx.x - head;
    store_one<D>(dx + at, grad_of(r, Vec<T>::one(x + at), at));
  }
}

// Blocks per row, by what a few rows take alone (us, 1 / 2 / 4 / 8 blocks): 1 row of 151936 13.0 / 8.8 / 6.1 / 5.1; 16 rows with 5
// alternatives 21.3 / 15.2 / 11.0 / 10.0; 64 of 128256 with 8 20.2 / 15.1 / 12.7 / 13.3; 150 without 16.0 / 13.3 / 13.1 / 15.0, with 8
// 24.4 / 21.0 / 22.4 / 27.5; 200 with 8 25.0 / 22.4 / 26.0 / 33.7.  From 300 rows on a second block only doubles what a block costs at its
// ends: 333 x 32003 with 5 13.3 / 18.8, 1024 x 128256 with 8 67 / 82.
static int scores_split(long long rows, int vocab) {
  int parts = 1;
  while (parts < 8 && 2 * rows * parts <= 3 * num_sms() && vocab / (2 * parts) >= 2048) parts *= 2;
  return parts;
}

void token_scores_fwd(const TokenScoreArgs& a, cudaStream_t s) {
  if (a.rows <= 0) return;
  if (a.vocab <= 0 || a.top_k < 0 || a.top_k > kTopMax || a.top_k > a.vocab) throw std::runtime_error("himuon token_scores: bad vocabulary or number of alternatives");
  const ScoreArgsDev p{a.logits, a.ids, a.log_probs, a.entropy, reinterpret_cast<float2*>(a.stats), a.top_log_probs, a.top_ids,
                       a.rows, a.ld, a.ignore, a.vocab, a.top_k};
  const int parts = scores_split(a.rows, a.vocab);
  if (a.rows * parts >= (1LL << 31)) throw std::runtime_error("himuon token_scores: too many rows for one launch");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.rows * parts));
  cfg.blockDim = dim3(NT);
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = parts; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  auto kern = a.logits_fp32 ? (a.top_k ? token_scores_kernel<float, true> : token_scores_kernel<float, false>)
                            : (a.top_k ? token_scores_kernel<__nv_bfloat16, true> : token_scores_kernel<__nv_bfloat16, false>);
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
  if (e != cudaSuccess) throw std::runtime_error(std::string("himuon token_scores launch failed: ") + cudaGetErrorString(e));
}

void token_scores_bwd(const TokenScoreArgs& a, cudaStream_t s) {
  if (a.rows <= 0) return;
  const ScoreGradDev p{a.logits, a.grad, a.ids, a.entropy, reinterpret_cast<const float2*>(a.stats), a.g_log_probs, a.g_entropy,
                       a.rows, a.ld, a.ld_grad, a.ignore, a.vocab};
  const int n = a.logits_fp32 ? 4 : 8;
  const long long per_row = (a.vocab / n + NT * SG_GROUPS - 1) / (NT * SG_GROUPS), blocks_per_row = per_row > 0 ? per_row : 1;
  if (a.vocab <= 0 || a.rows * blocks_per_row >= (1LL << 31)) throw std::runtime_error("himuon token_scores: gradient too large for one launch");
  const unsigned grid = static_cast<unsigned>(a.rows * blocks_per_row);
  const int b = static_cast<int>(blocks_per_row);
  if (a.logits_fp32) {
    if (a.grad_fp32) token_scores_grad_kernel<float, float><<<grid, NT, 0, s>>>(p, b);
    else token_scores_grad_kernel<float, __nv_bfloat16><<<grid, NT, 0, s>>>(p, b);
  } else {
    if (a.grad_fp32) throw std::runtime_error("himuon token_scores: bf16 logits have bf16 gradients");
    token_scores_grad_kernel<__nv_bfloat16, __nv_bfloat16><<<grid, NT, 0, s>>>(p, b);
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) throw std::runtime_error(std::string("himuon token_scores gradient launch failed: ") + cudaGetErrorString(e));
}

}  // namespace himuon
