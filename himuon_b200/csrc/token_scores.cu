// Log probability of given tokens, entropy and likeliest alternatives of rows of logits (bf16 or fp32), and the gradient
// that reaches the logits.
//
// With m = max x, d = x - m:   s = sum e^d,  t = sum d e^d,   log p_j = d_j - log s,   H = log s - t / s.
// Shifted by the maximum both sums have terms of one sign, so the entropy of a peaked row loses nothing to cancellation, and
// partial results merge: moving (m1, s1, t1) to a larger m scales s1 by f = e^(m1-m) and turns t1 into f (t1 + (m1-m) s1).
// Gradient, with the incoming g of log p_y and h of H:   dx_j = g [j = y] - p_j (g + h (log p_j + H)).
// A logit of -inf has p = 0 and no part in H.  A row of nothing but -inf has log p = -inf, H = 0 and no gradient.  An id equal to
// `ignore` has log p = 0 and passes no g on; an id outside the vocabulary has log p = NaN and passes none on either.
//
// One pass over the logits; their bytes bound both kernels.  A row goes to a cluster of 1 to 8 blocks, so that a few rows
// occupy the GPU as well (rule in scores_split()); the blocks' partial results meet in distributed shared memory.
// Likeliest alternatives: each warp keeps a sorted list of 32, one a lane, as 64-bit keys of value and inverted index, so that equal
// values go to the lower index.  What passes the list's k-th value is collected in shared memory and merged 32 at a time by a
// bitonic network; after the first few hundred elements of a row next to nothing passes.
#include <stdint.h>

#include "himuon.h"
#include "pair_common.cuh"
#include "sm100_common.cuh"

namespace himuon {

namespace {

constexpr int SC_THREADS = 256, SC_WARPS = SC_THREADS / 32;
constexpr float kLog2eS = 1.4426950408889634f;
constexpr float kFar = -1.0e4f;                   // d below this: e^d is 0 in fp32, and d * e^d has to be as well

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

struct Sums { float m, s, t; };
__device__ __forceinline__ Sums moved(const Sums& a, float m) {     // a's sums relative to m >= a.m
  if (a.m == -INFINITY) return Sums{m, a.s, a.t};                   // 0, or NaN
  const float d = fmaxf(a.m - m, kFar), f = exp2f(d * kLog2eS);
  return Sums{m, a.s * f, f * (a.t + d * a.s)};
}
__device__ __forceinline__ Sums merged(const Sums& a, const Sums& b) {
  const float m = fmaxf(a.m, b.m);
  const Sums x = moved(a, m), y = moved(b, m);
  return Sums{m, x.s + y.s, x.t + y.t};
}
template <int N>
__device__ __forceinline__ void take(Sums& a, const float (&x)[N]) {
  float mx = x[0];
#pragma unroll
  for (int i = 1; i < N; ++i) mx = fmaxf(mx, x[i]);
  if (mx > a.m) a = moved(a, mx);
  const float base = a.m == -INFINITY ? 0.f : a.m;    // nothing but -inf so far: d = -inf, e^d = 0
  const f32x2 nbase = pack2(-base, -base), l2e = pack2(kLog2eS, kLog2eS);
  f32x2 s = pack2(0.f, 0.f), t = s;
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const f32x2 d = add2(pack2(x[i], x[i + 1]), nbase);
    float d0, d1, y0, y1;
    unpack2(d, d0, d1);
    unpack2(mul2(d, l2e), y0, y1);
    const f32x2 e = pack2(exp2f(y0), exp2f(y1));
    s = add2(s, e);
    t = fma2(pack2(fmaxf(d0, kFar), fmaxf(d1, kFar)), e, t);
  }
  float a0, a1;
  unpack2(s, a0, a1);
  a.s += a0 + a1;
  unpack2(t, a0, a1);
  a.t += a0 + a1;
}

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
  Key kth;               // the k-th of the list, and its value
  float bar;
  int waiting;           // entries of `buf` in use, the same in all lanes
  Key* buf;              // 64 of this warp
  int lane, k;
  __device__ __forceinline__ void start(Key* b, int l, int k_) {
    best = 0; kth = 0; bar = -INFINITY; waiting = 0; buf = b; lane = l; k = k_;
  }
  __device__ __forceinline__ void flush() {
    __syncwarp();
    const Key x = lane < waiting ? buf[lane] : 0;
    const Key rest = lane + 32 < waiting ? buf[lane + 32] : 0;
    __syncwarp();
    buf[lane] = rest;
    best = merged_down(best, sorted_down(x, lane), lane);
    kth = __shfl_sync(0xffffffffu, best, k - 1);
    bar = kth ? key_value(kth) : -INFINITY;
    waiting = waiting > 32 ? waiting - 32 : 0;
  }
  // One value a lane (live lanes only); called by the whole warp.
  __device__ __forceinline__ void offer(float x, uint32_t index, bool live) {
    const Key key = key_of(x, index);
    const bool in = live && !(x < bar) && key > kth;
    const uint32_t who = __ballot_sync(0xffffffffu, in);
    if (who == 0) return;
    if (in) buf[waiting + __popc(who & ((1u << lane) - 1))] = key;
    waiting += __popc(who);
    if (waiting >= 32) flush();
  }
};

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

// Cluster = one row.  Block r of the cluster takes the r-th share of the row's whole 16-byte groups; what lies before the first
// group and behind the last goes to the first block.
template <typename T, bool TOP>
__global__ void __launch_bounds__(SC_THREADS)
token_scores_kernel(ScoreArgsDev p) {
  constexpr int N = Vec<T>::N, UN = TOP ? 2 : 4;
  __shared__ Sums s_sums[SC_WARPS];
  __shared__ Sums s_block;
  __shared__ Key s_buf[TOP ? SC_WARPS * 64 : 1];
  __shared__ Key s_list[TOP ? 32 : 1];

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

  Sums a{-INFINITY, 0.f, 0.f};
  TopList top;
  if (TOP) top.start(s_buf + warp * 64, lane, p.k);
  // every lane of a warp makes the same number of passes, with -inf where it is past the end
  const float none = -INFINITY;
  for (int g = g0 + warp * 32 * UN; g < g1; g += SC_THREADS * UN) {
    uint4 raw[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int i = g + u * 32 + lane;
      if (i < g1) raw[u] = __ldcs(body + i);
    }
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int i = g + u * 32 + lane;
      const bool live = i < g1;
      float v[N];
      Vec<T>::unpack(raw[u], v);
      if (live) take<N>(a, v);
      if (TOP) {
        bool any = false;
#pragma unroll
        for (int q = 0; q < N; ++q) any = any || !(v[q] < top.bar);
        if (__any_sync(0xffffffffu, live && any)) {
#pragma unroll 1
          for (int q = 0; q < N; ++q) {
            float xq = none;
#pragma unroll
            for (int r = 0; r < N; ++r) if (r == q) xq = v[r];
            top.offer(xq, static_cast<uint32_t>(head + i * N + q), live);
          }
        }
      }
    }
  }
  if (part == 0 && warp == 0) {                     // the ragged ends: fewer than 2 N elements
    const int tail0 = head + groups * N, loose = head + p.vocab - tail0;
    const bool live = lane < loose;
    const int at = lane < head ? lane : tail0 + lane - head;
    float v[2] = {none, none};
    if (live) v[0] = Vec<T>::one(x + at);
    if (live) take<2>(a, v);
    if (TOP) top.offer(v[0], static_cast<uint32_t>(at), live);
  }
  // lanes, warps, blocks
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Sums b{__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o), __shfl_xor_sync(0xffffffffu, a.t, o)};
    a = merged(a, b);
  }
  if (lane == 0) s_sums[warp] = a;
  if (TOP) {
    while (top.waiting > 0) top.flush();
    __syncwarp();
    top.buf[lane] = top.best;
  }
  __syncthreads();
  if (warp == 0) {
    a = s_sums[0];
    for (int w = 1; w < SC_WARPS; ++w) a = merged(a, s_sums[w]);
    if (TOP) {
      for (int w = 1; w < SC_WARPS; ++w) top.best = merged_down(top.best, s_buf[w * 64 + lane], lane);
    }
  }
  if (parts > 1) {                                  // uniform over the cluster
    if (warp == 0) {
      if (lane == 0) s_block = a;
      if (TOP) s_list[lane] = top.best;
    }
    __syncwarp();
    cluster_sync_all();
    if (part == 0 && warp == 0) {
      for (uint32_t r = 1; r < parts; ++r) {
        a = merged(a, load_remote(&s_block, r));
        if (TOP) top.best = merged_down(top.best, load_remote(&s_list[lane], r), lane);
      }
    }
    cluster_sync_all();                             // no block leaves while it is still read
  }
  if (part == 0 && warp == 0) {
    const bool empty = a.s == 0.f;                  // nothing but -inf (a NaN makes s NaN)
    const float m = empty ? 0.f : a.m;
    const float log_s = empty ? INFINITY : static_cast<float>(log(static_cast<double>(a.s)));   // (logf is the approximate one in this build)
    if (lane == 0) {
      const long long y = p.ids[row];
      float lp = 0.f;
      if (y != p.ignore) lp = y >= 0 && y < p.vocab ? (Vec<T>::one(x + y) - m) - log_s : __uint_as_float(0x7FFFFFFFu);
      p.log_probs[row] = lp;
      p.entropy[row] = empty ? 0.f : log_s - a.t / a.s;
      if (p.stats) p.stats[row] = make_float2(m, log_s);
    }
    if (TOP && lane < p.k) {
      p.top_log_probs[row * p.k + lane] = (key_value(top.best) - m) - log_s;
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

// dx of N logits from column `at` on.
template <int N>
__device__ __forceinline__ void grad_of(const float (&x)[N], float (&d)[N], int at, float m, float log_s, float c0, float h, float g, long long y) {
#pragma unroll
  for (int q = 0; q < N; ++q) {
    const float lp = (x[q] - m) - log_s, e = exp2f(lp * kLog2eS);
    d[q] = -e * fmaf(h, fmaxf(lp, kFar), c0);
    if (at + q == y) d[q] += g;
  }
}
// T: logits, D: gradient.  Rows that share the offset from 16 bytes with the gradient's are read and written in 16-byte groups of
// logits; others element by element.
constexpr int SG_GROUPS = 4;                        // 16-byte groups of logits a thread takes
template <typename T, typename D>
__global__ void __launch_bounds__(SC_THREADS)
token_scores_grad_kernel(ScoreGradDev p, int blocks_per_row) {
  constexpr int N = Vec<T>::N;
  const long long row = blockIdx.x / blocks_per_row;
  const int piece = static_cast<int>(blockIdx.x - row * blocks_per_row);
  const T* x = reinterpret_cast<const T*>(p.logits) + row * p.ld;
  D* dx = reinterpret_cast<D*>(p.grad) + row * p.ld_grad;
  const float2 st = p.stats[row];
  const long long id = p.ids[row];
  const bool counted = id != p.ignore && id >= 0 && id < p.vocab;
  const long long y = counted && st.y != INFINITY ? id : -1;             // (INFINITY: a row of nothing but -inf)
  const float g = counted && p.g_log_probs ? p.g_log_probs[row] : 0.f;
  const float h = p.g_entropy ? p.g_entropy[row] : 0.f, c0 = fmaf(h, p.entropy[row], g);

  int head = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / static_cast<int>(sizeof(T));
  if (head > p.vocab) head = p.vocab;
  const bool wide = (reinterpret_cast<uintptr_t>(dx + head) & (N * sizeof(D) - 1) & 15) == 0;
  const int groups = (p.vocab - head) / N;
#pragma unroll
  for (int u = 0; u < SG_GROUPS; ++u) {
    const int i = (piece * SG_GROUPS + u) * SC_THREADS + static_cast<int>(threadIdx.x);
    if (i >= groups) break;
    const int at = head + i * N;
    float v[N], d[N];
    Vec<T>::unpack(__ldcs(reinterpret_cast<const uint4*>(x + head) + i), v);
    grad_of<N>(v, d, at, st.x, st.y, c0, h, g, y);
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
    const float v[1] = {Vec<T>::one(x + at)};
    float d[1];
    grad_of<1>(v, d, at, st.x, st.y, c0, h, g, y);
    store_one<D>(dx + at, d[0]);
  }
}

// Blocks per row: doubled while the launch would still not fill the GPU and a share keeps a few thousand logits.
static int scores_split(long long rows, int vocab) {
  int parts = 1;
  while (parts < 8 && rows * parts < 4LL * num_sms() && vocab / (2 * parts) >= 2048) parts *= 2;
  return parts;
}

void token_scores_fwd(const TokenScoreArgs& a, cudaStream_t s) {
  if (a.rows <= 0) return;
  const ScoreArgsDev p{a.logits, a.ids, a.log_probs, a.entropy, reinterpret_cast<float2*>(a.stats), a.top_log_probs, a.top_ids,
                       a.rows, a.ld, a.ignore, a.vocab, a.top_k};
  const int parts = scores_split(a.rows, a.vocab);
  if (a.vocab <= 0 || a.top_k < 0 || a.top_k > kTopMax || a.top_k > a.vocab) throw std::runtime_error("himuon token_scores: bad vocabulary or number of alternatives");
  if (a.rows * parts >= (1LL << 31)) throw std::runtime_error("himuon token_scores: too many rows for one launch");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.rows * parts));
  cfg.blockDim = dim3(SC_THREADS);
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
  const long long per_row = (a.vocab / n + SC_THREADS * SG_GROUPS - 1) / (SC_THREADS * SG_GROUPS), blocks_per_row = per_row > 0 ? per_row : 1;
  if (a.vocab <= 0 || a.rows * blocks_per_row >= (1LL << 31)) throw std::runtime_error("himuon token_scores: gradient too large for one launch");
  const unsigned grid = static_cast<unsigned>(a.rows * blocks_per_row);
  const int b = static_cast<int>(blocks_per_row);
  if (a.logits_fp32) {
    if (a.grad_fp32) token_scores_grad_kernel<float, float><<<grid, SC_THREADS, 0, s>>>(p, b);
    else token_scores_grad_kernel<float, __nv_bfloat16><<<grid, SC_THREADS, 0, s>>>(p, b);
  } else {
    if (a.grad_fp32) throw std::runtime_error("himuon token_scores: bf16 logits have bf16 gradients");
    token_scores_grad_kernel<__nv_bfloat16, __nv_bfloat16><<<grid, SC_THREADS, 0, s>>>(p, b);
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) throw std::runtime_error(std::string("himuon token_scores gradient launch failed: ") + cudaGetErrorString(e));
}

}  // namespace himuon
