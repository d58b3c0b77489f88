// Rotary positions: the first `rotary_dim` values of every head are pairs (a, b), turned by the angle of their position,
//     a' = c a - s b,   b' = c b + s a,   c = m cos(pos f_i), s = m sin(pos f_i);
// the values behind them pass through.  Pairs are (i, i + rotary_dim / 2) or, interleaved, (2i, 2i + 1).  The gradient is the same with -s.
//
// Angles.  fp32 angles of far positions are off by pos * 2^-24 of a radian and more (0.008 at 131071).  Here a frequency is a whole
// number of 2^-64 turns a position, so that pos * f modulo 2^64 is the angle's place within its turn, exact to pos * 2^-65 of a turn at any
// position, with no table to make, keep or read.  Its upper 32 bits go to sincospif.
//
// Bounded by memory: every value is read and written once.  A block has some rows, of all heads or of a share of them.  Its threads ask for their first
// values, work out a sine and cosine each while those are on their way, and leave them in shared memory for all the heads; then they take pairs of vectors of 16
// bytes (a's and b's of the same pairs, or two that pass through), two pairs at a time.  With every thread working out the eight sines of its own vectors, for a
// quarter of the heads: 4071 rows of 20 heads of 64 7.1 us.
#include "rotary.h"

#include <algorithm>

#include "himuon.h"
#include "sm100_common.cuh"

namespace himuon {

namespace {

constexpr int ROT_WAVES = 1024;      // sines and cosines that a block has room for

struct RotaryDev {
  RotaryArgs a;
  int units;                 // pairs of vectors in a head
  int rows, heads;           // of a block
  int lanes;                 // rotary_any_kernel: heads that neighbouring threads take, of the `heads`
  long long threads;         // rows * lanes * units
};

// (m cos, m sin).  As a float, a place next to half a turn is off by 2^-26 of a turn, and its sine, which is near 0, by 9e-8: nothing beside the rounding of
// bf16 results, so that they go without what fp32 ones need (4096 rows of 20 heads of 128 8.1 us, 8.4 with it).
template <typename T>
__device__ __forceinline__ float2 wave(const RotaryArgs& a, long long pos, int i) {
  const unsigned long long t = static_cast<unsigned long long>(pos) * a.turns[i];
  float s, c;
  if constexpr (sizeof(T) == 2) {
    sincospif(static_cast<float>(static_cast<int>(t >> 32)) * 0x1p-31f, &s, &c);      // (2^32 is a turn, pi half of one)
  } else {
    // what is left from the nearest quarter of a turn, and the bits of it that a float does not hold
    const uint32_t place = static_cast<uint32_t>((t + 0x80000000ull) >> 32), quarters = place + 0x20000000u;      // (bits 30 and 31)
    const int rest = static_cast<int>(place - (quarters & 0xC0000000u));
    const float near = __int2float_rn(rest), low = static_cast<float>(rest - __float2int_rn(near)) * 1.4629180792671596e-9f;      // (2 pi / 2^32)
    float sn, cn;
    sincospif(near * 0x1p-31f, &sn, &cn);
    const float sl = fmaf(cn, low, sn), cl = fmaf(-sn, low, cn);
    s = quarters & 0x40000000u ? cl : sl;              // a quarter on: sine and cosine change places, and one of them its sign
    c = quarters & 0x40000000u ? sl : cl;
    if (quarters & 0x80000000u) s = -s;
    if ((quarters ^ (quarters << 1)) & 0x80000000u) c = -c;
  }
  return make_float2(c * a.cos_factor, s * a.sin_factor);
}
// One pair, with the same roundings in every kernel.
__device__ __forceinline__ void turn(const float2& w, float& a, float& b) {
  const float was = a;
  a = fmaf(w.x, was, -__fmul_rn(w.y, b));
  b = fmaf(w.x, b, __fmul_rn(w.y, was));
}
__device__ __forceinline__ long long position(const RotaryArgs& a, long long row) { return a.positions ? a.positions[row] : row % a.seq_len; }

template <typename T> struct Vec;
template <> struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void get(const uint4& v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[2 * i] = bf16_lo(w[i]); f[2 * i + 1] = bf16_hi(w[i]); }
  }
  static __device__ __forceinline__ uint4 put(const float (&f)[8]) {
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  }
};
template <> struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void get(const uint4& v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ uint4 put(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};

// Whole vectors: heads of whole vectors, rows on 16-byte boundaries, and no vector with both halves of a pair unless interleaved.
template <typename T, bool INTERLEAVED>
__global__ void __launch_bounds__(256) rotary_vec_kernel(RotaryDev p) {
  constexpr int N = Vec<T>::N, BATCH = 2;
  __shared__ float2 s_wave[ROT_WAVES];
  const RotaryArgs& a = p.a;
  const int vecs = a.head_dim / N, turned = a.rotary_dim / N, pairs = a.rotary_dim / 2;
  const long long row0 = static_cast<long long>(blockIdx.x) * p.rows;
  const int h0 = static_cast<int>(blockIdx.y) * p.heads, nh = min(p.heads, a.heads - h0), nr = static_cast<int>(min(static_cast<long long>(p.rows), a.rows - row0));
  const int items = nr * nh * p.units;
  struct Item {
    uint4 q0, q1;
    long long to;            // of the head, in the result
    int v0, v1, row;         // its two vectors, and the row
    bool there, second, turn0, turn1;
  };
  auto fetch = [&](int i, Item& it) {
    it.there = i < items;
    if (!it.there) return;
    const int unit = i % p.units, rest = i / p.units, h = h0 + rest % nh;
    it.row = rest / nh;
    if (INTERLEAVED) {
      it.v0 = unit; it.v1 = unit + p.units;
      it.turn0 = it.v0 < turned; it.turn1 = it.v1 < turned;
    } else if (unit < turned / 2) {
      it.v0 = unit; it.v1 = unit + turned / 2;
      it.turn0 = it.turn1 = true;
    } else {
      it.v0 = unit + turned / 2; it.v1 = it.v0 + (vecs - turned + 1) / 2;
      it.turn0 = it.turn1 = false;
    }
    it.second = it.v1 < vecs;
    it.to = (row0 + it.row) * a.ld_y + static_cast<long long>(h) * a.head_dim;
    const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.x) + (row0 + it.row) * a.ld_x + static_cast<long long>(h) * a.head_dim);
    it.q0 = src[it.v0];
    it.q1 = it.second ? src[it.v1] : make_uint4(0, 0, 0, 0);
  };
  auto finish = [&](Item& it) {
    if (!it.there) return;
    if (it.turn0) {
      const float2* w = s_wave + it.row * pairs;
      float f0[N], f1[N];
      Vec<T>::get(it.q0, f0);
      Vec<T>::get(it.q1, f1);
      if (INTERLEAVED) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
          turn(w[it.v0 * (N / 2) + i], f0[2 * i], f0[2 * i + 1]);
          if (it.turn1) turn(w[it.v1 * (N / 2) + i], f1[2 * i], f1[2 * i + 1]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) turn(w[it.v0 * N + i], f0[i], f1[i]);
      }
      it.q0 = Vec<T>::put(f0);
      if (!INTERLEAVED || it.turn1) it.q1 = Vec<T>::put(f1);       // (what passes through keeps its bits)
    }
    uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.y) + it.to);
    dst[it.v0] = it.q0;
    if (it.second) dst[it.v1] = it.q1;
  };
  Item batch[BATCH];
#pragma unroll
  for (int b = 0; b < BATCH; ++b) fetch(threadIdx.x + b * 256, batch[b]);
  for (int i = threadIdx.x; i < nr * pairs; i += 256) {
    const int r = i / pairs;
    s_wave[i] = wave<T>(a, position(a, row0 + r), i - r * pairs);
  }
  __syncthreads();
  for (int at = threadIdx.x;; ) {
#pragma unroll
    for (int b = 0; b < BATCH; ++b) finish(batch[b]);
    at += BATCH * 256;
    if (at >= items) break;
#pragma unroll
    for (int b = 0; b < BATCH; ++b) fetch(at + b * 256, batch[b]);
  }
}

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// Any even rotary_dim, any row stride: a thread has one pair, or one value that passes through, of all the heads.
template <typename T>
__global__ void __launch_bounds__(256) rotary_any_kernel(RotaryDev p) {
  const RotaryArgs& a = p.a;
  const long long id = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  if (id >= p.threads) return;
  const int unit = static_cast<int>(id % p.units);
  const long long rest = id / p.units;
  const int first = static_cast<int>(rest % p.lanes), half = a.rotary_dim / 2;
  const long long row = rest / p.lanes;
  const T* x = reinterpret_cast<const T*>(a.x) + row * a.ld_x;
  T* y = reinterpret_cast<T*>(a.y) + row * a.ld_y;
  if (unit >= half) {
    for (int h = first; h < a.heads; h += p.lanes) {
      const long long at = static_cast<long long>(h) * a.head_dim + half + unit;
      y[at] = x[at];
    }
    return;
  }
  const float2 w = wave<T>(a, position(a, row), unit);
  const int i0 = a.interleaved ? 2 * unit : unit, i1 = a.interleaved ? 2 * unit + 1 : unit + half;
  for (int h = first; h < a.heads; h += p.lanes) {
    const long long at = static_cast<long long>(h) * a.head_dim;
    float f0 = as_float(x[at + i0]), f1 = as_float(x[at + i1]);
    turn(w, f0, f1);
    put(y + at + i0, f0);
    put(y + at + i1, f1);
  }
}

template <typename T>
void launch(const RotaryArgs& a, cudaStream_t s) {
  constexpr int N = Vec<T>::N;
  auto grid16 = [](const void* p, long long ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % N == 0; };
  const bool whole = a.head_dim % N == 0 && a.rotary_dim % (a.interleaved ? N : 2 * N) == 0 && a.rotary_dim / 2 <= ROT_WAVES && grid16(a.x, a.ld_x) && grid16(a.y, a.ld_y);
  RotaryDev p{};
  p.a = a;
  if (whole) {
    const int pairs = std::max(a.rotary_dim / 2, 1);
    p.units = (a.head_dim / N + 1) / 2;
    // as many rows as there are sines for the threads, but four blocks a SM, if need be with a share of the heads each
    const long long want = 4LL * num_sms();
    p.rows = static_cast<int>(std::max(1LL, std::min<long long>(256 / pairs, a.rows / want)));
    const long long blocks = (a.rows + p.rows - 1) / p.rows, shares = std::max(1LL, std::min<long long>(want / blocks, a.heads * p.units / 64));
    p.heads = static_cast<int>((a.heads + shares - 1) / shares);
    if (blocks >= (1LL << 31)) throw std::runtime_error("himuon rotary: too many rows for one launch");
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>((a.heads + p.heads - 1) / p.heads));
    if (a.interleaved) rotary_vec_kernel<T, true><<<grid, 256, 0, s>>>(p);
    else rotary_vec_kernel<T, false><<<grid, 256, 0, s>>>(p);
  } else {
    p.units = a.head_dim - a.rotary_dim / 2;
    p.lanes = std::min(a.heads, 4);
    p.threads = a.rows * p.lanes * p.units;
    const long long blocks = (p.threads + 255) / 256;
    if (blocks >= (1LL << 31)) throw std::runtime_error("himuon rotary: too many rows for one launch");
    rotary_any_kernel<T><<<static_cast<int>(blocks), 256, 0, s>>>(p);
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) throw std::runtime_error(std::string("himuon rotary launch failed: ") + cudaGetErrorString(e));
}

}  // namespace

void rotary(const RotaryArgs& a, cudaStream_t s) {
  if (a.rows <= 0 || a.heads <= 0 || a.head_dim <= 0) return;
  if (a.rotary_dim < 0 || a.rotary_dim % 2 || a.rotary_dim > a.head_dim || (a.positions == nullptr && a.seq_len <= 0)) throw std::runtime_error("himuon rotary: bad sizes");
  if (a.fp32) launch<float>(a, s);
  else launch<__nv_bfloat16>(a, s);
}

}  // namespace himuon
