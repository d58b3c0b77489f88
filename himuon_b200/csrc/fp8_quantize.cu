// Matrices in 8 bits: e4m3 values and a power of two for each block of (1, 128) or (128, 128) of them.
//
//   scale = the least 2^k with max |x| <= 448 * 2^k (1 where the block holds nothing but zeros, 2^-110 at the least),  q = rn_e4m3(x / scale)
//
// A power of two makes the division exact, so that q has one rounding of x (2^-4 of it at most, or 2^-10 of the scale) and no value next to a tie
// hangs on the rounding of a quotient; it costs up to one bit of range at the lower end, of 17.  A value that is not finite becomes NaN and has no part
// in its block's scale.  Below 2^-110 * 2^-10 there is nothing left, also not what this build's arithmetic would flush.
//
// Bounded by memory: every value is read once, for all the copies that are wanted.  Where a row's blocks are all that is wanted, 16 threads take a block of
// 128 values.  Otherwise a block of 256 threads has 128 x 128 values, 8 x 8 a thread, and turns them around in shared memory; it holds them as they
// came (a bf16 pair in a register), since as fp32 they left room for one block to an SM (8192 x 9728 by rows 190 us so).
#include <cuda_fp8.h>

#include "fp8.h"
#include "himuon.h"
#include "sm100_common.cuh"

namespace himuon {

namespace {

constexpr int QT = 128;              // rows and columns of a block

// k of the scale of a block whose largest finite value has these bits.
__device__ __forceinline__ int scale_exponent(uint32_t bits) {
  if (bits == 0) return 0;
  // 448 = 1.75 * 2^8
  const int k = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return k < -110 ? -110 : k;
}
__device__ __forceinline__ float power_of_two(int k) { return __uint_as_float(static_cast<uint32_t>(k + 127) << 23); }
__device__ __forceinline__ uint32_t two(float a, float b) { return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3); }
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) { return two(a, b) | (two(c, d) << 16); }
__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

constexpr uint32_t kInfinite = 0x7F800000u;

// Eight neighbouring values as they came.
template <typename T> struct Eight {
  static constexpr int W = sizeof(T) * 2;
  uint32_t w[W];
  // `valid` of them (none: zeros); `whole`: all eight, on a 16-byte boundary.
  __device__ __forceinline__ void load(const T* p, int valid, bool whole) {
    if (whole) {
#pragma unroll
      for (int i = 0; i < W / 4; ++i) reinterpret_cast<uint4*>(w)[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i) w[i] = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < valid) {
          if constexpr (sizeof(T) == 2) w[j / 2] |= static_cast<uint32_t>(__bfloat16_as_ushort(p[j])) << (16 * (j & 1));
          else w[j] = __float_as_uint(p[j]);
        }
    }
  }
  __device__ __forceinline__ float at(int j) const {
    if constexpr (sizeof(T) == 2) return (j & 1) ? bf16_hi(w[j / 2]) : bf16_lo(w[j / 2]);
    else return __uint_as_float(w[j]);
  }
  // Bits of the largest absolute value, as of an fp32 number; of kInfinite or more where one is not finite.
  __device__ __forceinline__ uint32_t largest() const {
    uint32_t m = 0;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < W; ++i) m = __vmaxu2(m, w[i] & 0x7FFF7FFFu);
      return max(m << 16, m & 0xFFFF0000u);
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i) m = max(m, w[i] & 0x7FFFFFFFu);
      return m;
    }
  }
  // The same of the eight columns of eight rows.
  static __device__ __forceinline__ void largest_of_columns(const Eight (&rows)[8], uint32_t (&out)[8]) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < W; ++i) {
        uint32_t m = 0;
#pragma unroll
        for (int r = 0; r < 8; ++r) m = __vmaxu2(m, rows[r].w[i] & 0x7FFF7FFFu);
        out[2 * i] = m << 16;
        out[2 * i + 1] = m & 0xFFFF0000u;
      }
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i)
#pragma unroll
        for (int r = 0; r < 8; ++r) out[i] = max(out[i], rows[r].w[i] & 0x7FFFFFFFu);
    }
  }
  // largest() of the finite ones.
  __device__ __forceinline__ uint32_t largest_finite() const {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t b = __float_as_uint(at(j)) & 0x7FFFFFFFu;
      m = max(m, b < kInfinite ? b : 0u);
    }
    return m;
  }
  __device__ __forceinline__ uint2 quantized(float by) const {
    return make_uint2(pack4(at(0) * by, at(1) * by, at(2) * by, at(3) * by), pack4(at(4) * by, at(5) * by, at(6) * by, at(7) * by));
  }
  // Infinities become NaN.
  __device__ __forceinline__ void mark() {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < W; ++i) {
        if ((w[i] & 0x7F80u) == 0x7F80u) w[i] |= 0x7Fu;
        if ((w[i] & 0x7F800000u) == kInfinite) w[i] |= 0x7F0000u;
      }
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i)
        if ((w[i] & kInfinite) == kInfinite) w[i] |= 0x7FFFFFu;
    }
  }
};

template <int LANES>
__device__ __forceinline__ uint32_t largest_of(uint32_t m) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}

// Of eight values in each of 16 lanes, the largest of all lanes: of the value tc / 2 in lane tc.  (Lanes halve what they have as they go: 8 shuffles, not 32.)
__device__ __forceinline__ uint32_t largest_of_rows(const uint32_t (&m)[8], int tc) {
  uint32_t a[4], b[2];
  const bool h = tc & 8, q = tc & 4, e = tc & 2;
#pragma unroll
  for (int i = 0; i < 4; ++i) a[i] = max(h ? m[i + 4] : m[i], __shfl_xor_sync(0xffffffffu, h ? m[i] : m[i + 4], 8));
#pragma unroll
  for (int i = 0; i < 2; ++i) b[i] = max(q ? a[i + 2] : a[i], __shfl_xor_sync(0xffffffffu, q ? a[i] : a[i + 2], 4));
  const uint32_t c = max(e ? b[1] : b[0], __shfl_xor_sync(0xffffffffu, e ? b[0] : b[1], 2));
  return max(c, __shfl_xor_sync(0xffffffffu, c, 1));
}

// Rows by themselves: 16 threads take RUN neighbouring blocks of a row; the 16 rows of a block of threads have their scales one behind the other, as products read them
// (8192 x 9728 49.4 us; with a run and the next of a row side by side 52.5, with blocks that stay and take run after run 60).
constexpr int RUN = 4;
template <typename T>
__global__ void __launch_bounds__(256) fp8_quantize_rows_kernel(Fp8QuantizeArgs a, int runs, int blocks_c, int aligned) {
  launch_dependents();
  const int group = static_cast<int>(blockIdx.x) / runs, b0 = (static_cast<int>(blockIdx.x) - group * runs) * RUN, lane = threadIdx.x & 15;
  const bool mine = group * 16LL + (threadIdx.x >> 4) < a.rows;      // (all 32 lanes meet in the shuffles)
  const long long row = mine ? group * 16LL + (threadIdx.x >> 4) : 0;
  const Fp8Out& o = a.straight;
  Eight<T> v[RUN];
#pragma unroll
  for (int i = 0; i < RUN; ++i) {
    const long long c = static_cast<long long>(b0 + i) * QT + lane * 8;
    const int valid = mine && c < a.cols ? static_cast<int>(a.cols - c < 8 ? a.cols - c : 8) : 0;
    v[i].load(reinterpret_cast<const T*>(a.x) + row * a.ld + c, valid, valid == 8 && aligned);
  }
#pragma unroll
  for (int i = 0; i < RUN; ++i) {
    uint32_t m = largest_of<16>(v[i].largest());
    if (__any_sync(0xffffffffu, m >= kInfinite)) {
      m = largest_of<16>(v[i].largest_finite());
      v[i].mark();
    }
    const int k = scale_exponent(m);
    const long long c = static_cast<long long>(b0 + i) * QT + lane * 8;
    if (mine && b0 + i < blocks_c) {
      if (c < o.ld) *reinterpret_cast<uint2*>(static_cast<uint8_t*>(o.values) + row * o.ld + c) = v[i].quantized(power_of_two(-k));      // (zeros behind the last column)
      if (lane == 0) o.scales[row * o.scale_row + (b0 + i) * o.scale_col] = power_of_two(k);
    }
  }
}

// Any copies: STRAIGHT and TURNED are the rows of their blocks, or 0 for none.
template <typename T, int STRAIGHT, int TURNED>
__global__ void __launch_bounds__(256) fp8_quantize_kernel(Fp8QuantizeArgs a, int tiles_c, int aligned) {
  launch_dependents();
  __shared__ uint32_t s_col[QT];
  __shared__ uint32_t s_all;
  __shared__ uint2 s_turned[TURNED ? QT * 16 : 1];     // [column][group of 8 rows, swizzled]
  const int tr = threadIdx.x >> 4, tc = threadIdx.x & 15;
  const long long rblk = blockIdx.x / tiles_c, cblk = blockIdx.x - rblk * tiles_c;
  const long long r0 = rblk * QT + tr * 8, c0 = cblk * QT + tc * 8;
  Eight<T> v[8];
  const int valid = a.cols <= c0 ? 0 : static_cast<int>(a.cols - c0 < 8 ? a.cols - c0 : 8);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const bool in = r0 + i < a.rows;
    v[i].load(reinterpret_cast<const T*>(a.x) + (r0 + i) * a.ld + c0, in ? valid : 0, in && valid == 8 && aligned);
  }
  constexpr bool WHOLE = STRAIGHT == QT || TURNED == QT;
  if (TURNED == 1 && threadIdx.x < QT) s_col[threadIdx.x] = 0;
  if (WHOLE && threadIdx.x == 0) s_all = 0;
  uint32_t row_max[8], m_all = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m_all = max(m_all, row_max[i] = v[i].largest());
  const bool finite = !__syncthreads_or(m_all >= kInfinite);
  if (!finite) {
    m_all = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m_all = max(m_all, row_max[i] = v[i].largest_finite());
  }
  if constexpr (WHOLE) {
    const uint32_t m = largest_of<32>(m_all);
    if ((threadIdx.x & 31) == 0) atomicMax(&s_all, m);
  }
  if constexpr (TURNED == 1) {
    uint32_t col_max[8] = {};
    if (finite) {
      Eight<T>::largest_of_columns(v, col_max);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t b = __float_as_uint(v[i].at(j)) & 0x7FFFFFFFu;
          col_max[j] = max(col_max[j], b < kInfinite ? b : 0u);
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t m = max(col_max[j], __shfl_xor_sync(0xffffffffu, col_max[j], 16));
      if ((threadIdx.x & 16) == 0) atomicMax(&s_col[tc * 8 + j], m);
    }
  }
  if (WHOLE || TURNED) __syncthreads();
  const int all = WHOLE ? scale_exponent(s_all) : 0;
  if constexpr (TURNED == 1) {                         // (once for each column, not by all threads that have values of it)
    if (threadIdx.x < QT) {
      const int k = scale_exponent(s_col[threadIdx.x]);
      if (cblk * QT + threadIdx.x < a.cols) a.turned.scales[(cblk * QT + threadIdx.x) * a.turned.scale_row + rblk * a.turned.scale_col] = power_of_two(k);
      s_col[threadIdx.x] = __float_as_uint(power_of_two(-k));
    }
  }
  if (!finite) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i].mark();
  }
  if constexpr (STRAIGHT != 0) {
    const Fp8Out& o = a.straight;
    int k_own = 0;
    if constexpr (STRAIGHT == 1) {
      k_own = scale_exponent(largest_of_rows(row_max, tc));
      if ((tc & 1) == 0 && r0 + tc / 2 < a.rows) o.scales[(r0 + tc / 2) * o.scale_row + cblk * o.scale_col] = power_of_two(k_own);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int k = STRAIGHT == QT ? all : __shfl_sync(0xffffffffu, k_own, (threadIdx.x & 16) | (2 * i));
      if (r0 + i < a.rows && c0 < o.ld)                // (behind the last column, up to the row's end, are zeros)
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(o.values) + (r0 + i) * o.ld + c0) = v[i].quantized(power_of_two(-k));
    }
    if (threadIdx.x == 0 && STRAIGHT == QT) o.scales[rblk * o.scale_row + cblk * o.scale_col] = power_of_two(all);
  }
  if constexpr (TURNED != 0) {
    const Fp8Out& o = a.turned;
    if (TURNED == 1) __syncthreads();                  // (s_col has factors)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = tc * 8 + j;
      const float by = TURNED == QT ? power_of_two(-all) : __uint_as_float(s_col[c]);
      s_turned[c * 16 + (tr ^ tc)] = make_uint2(pack4(v[0].at(j) * by, v[1].at(j) * by, v[2].at(j) * by, v[3].at(j) * by),
                                                pack4(v[4].at(j) * by, v[5].at(j) * by, v[6].at(j) * by, v[7].at(j) * by));
    }
    if (TURNED == QT && threadIdx.x == 0) o.scales[cblk * o.scale_row + rblk * o.scale_col] = power_of_two(all);
    __syncthreads();
    const long long at = rblk * QT + tc * 8;           // now 16 threads for the 128 rows of a column
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = i * 16 + tr;
      if (cblk * QT + c < a.cols && at < o.ld)
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(o.values) + (cblk * QT + c) * o.ld + at) = s_turned[c * 16 + (tc ^ (c >> 3))];
    }
  }
}

// Four values a thread and group, so that 32 threads write 512 bytes in a row; GROUPS groups of a row whose loads are under way together.
constexpr int GROUPS = 4;
template <typename T>
__global__ void __launch_bounds__(256) fp8_dequantize_kernel(Fp8Matrix m, T* out, long long ld_out, int pieces, int fast) {
  const long long row = blockIdx.x / pieces;
  const int col0 = (static_cast<int>(blockIdx.x - row * pieces) * GROUPS * 256 + static_cast<int>(threadIdx.x)) * 4;
  const uint8_t* src = static_cast<const uint8_t*>(m.values) + row * m.ld;
  const float* scales = m.scales + (m.block_rows == 1 ? row : row / QT) * m.scale_row;
  T* dst = out + row * ld_out;
  uint32_t q[GROUPS];
  float scale[GROUPS];
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) {
    const int col = col0 + g * 1024;
    q[g] = 0;
    scale[g] = 0.f;
    if (col < m.cols) {
      scale[g] = scales[(col / QT) * m.scale_col];
      if (fast) {
        q[g] = __ldcs(reinterpret_cast<const uint32_t*>(src + col));
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (col + j < m.cols) q[g] |= static_cast<uint32_t>(src[col + j]) << (8 * j);
      }
    }
  }
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) {
    const int col = col0 + g * 1024;
    if (col >= m.cols) break;
    const float2 lo = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(q[g] & 0xFFFFu), __NV_E4M3)));
    const float2 hi = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(q[g] >> 16), __NV_E4M3)));
    const float f[4] = {lo.x * scale[g], lo.y * scale[g], hi.x * scale[g], hi.y * scale[g]};
    if (fast) {
      if constexpr (sizeof(T) == 4) __stcs(reinterpret_cast<float4*>(dst + col), make_float4(f[0], f[1], f[2], f[3]));
      else __stcs(reinterpret_cast<uint2*>(dst + col), make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3])));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (col + j < m.cols) put(dst + col + j, f[j]);
    }
  }
}

void check(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) throw std::runtime_error(std::string("himuon ") + what + " launch failed: " + cudaGetErrorString(e));
}

template <typename T>
void launch_quantize(const Fp8QuantizeArgs& a, int tiles, int tiles_c, int runs, int groups, cudaStream_t s) {
  const int aligned = reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && a.ld % (16 / static_cast<int>(sizeof(T))) == 0;
  const int straight = a.straight.values ? a.straight.block_rows : 0, turned = a.turned.values ? a.turned.block_rows : 0;
  if (straight == 1 && !turned) fp8_quantize_rows_kernel<T><<<groups * runs, 256, 0, s>>>(a, runs, tiles_c, aligned);
  else if (straight == QT && !turned) fp8_quantize_kernel<T, QT, 0><<<tiles, 256, 0, s>>>(a, tiles_c, aligned);
  else if (!straight && turned == 1) fp8_quantize_kernel<T, 0, 1><<<tiles, 256, 0, s>>>(a, tiles_c, aligned);
  else if (!straight && turned == QT) fp8_quantize_kernel<T, 0, QT><<<tiles, 256, 0, s>>>(a, tiles_c, aligned);
  else if (straight == 1 && turned == 1) fp8_quantize_kernel<T, 1, 1><<<tiles, 256, 0, s>>>(a, tiles_c, aligned);
  else if (straight == 1 && turned == QT) fp8_quantize_kernel<T, 1, QT><<<tiles, 256, 0, s>>>(a, tiles_c, aligned);
  else if (straight == QT && turned == QT) fp8_quantize_kernel<T, QT, QT><<<tiles, 256, 0, s>>>(a, tiles_c, aligned);
  else throw std::runtime_error("himuon fp8_quantize: no such pair of copies");
}

}  // namespace

void fp8_quantize(const Fp8QuantizeArgs& a, cudaStream_t s) {
  if (a.rows <= 0 || a.cols <= 0) return;
  for (const Fp8Out* o : {&a.straight, &a.turned})
    if (o->values && ((o->block_rows != 1 && o->block_rows != QT) || o->ld % 16 || reinterpret_cast<uintptr_t>(o->values) % 16))
      throw std::runtime_error("himuon fp8_quantize: blocks of 1 or 128 rows, rows of multiples of 16 bytes");
  const long long tiles_c = (a.cols + QT - 1) / QT, tiles = (a.rows + QT - 1) / QT * tiles_c, runs = (tiles_c + RUN - 1) / RUN, groups = (a.rows + 15) / 16;
  if (tiles >= (1LL << 31) || groups * runs >= (1LL << 31)) throw std::runtime_error("himuon fp8_quantize: matrix too large for one launch");
  if (a.fp32) launch_quantize<float>(a, static_cast<int>(tiles), static_cast<int>(tiles_c), static_cast<int>(runs), static_cast<int>(groups), s);
  else launch_quantize<__nv_bfloat16>(a, static_cast<int>(tiles), static_cast<int>(tiles_c), static_cast<int>(runs), static_cast<int>(groups), s);
  check("fp8_quantize");
}

void fp8_dequantize(const Fp8Matrix& m, void* out, long long ld_out, int out_fp32, cudaStream_t s) {
  if (m.rows <= 0 || m.cols <= 0) return;
  const int fast = m.cols % 4 == 0 && m.ld % 4 == 0 && reinterpret_cast<uintptr_t>(m.values) % 4 == 0 && ld_out % 4 == 0 &&
                   reinterpret_cast<uintptr_t>(out) % 16 == 0;
  const int pieces = (m.cols + GROUPS * 1024 - 1) / (GROUPS * 1024);
  const long long blocks = static_cast<long long>(m.rows) * pieces;
  if (blocks >= (1LL << 31)) throw std::runtime_error("himuon fp8_dequantize: matrix too large for one launch");
  if (out_fp32) fp8_dequantize_kernel<float><<<static_cast<int>(blocks), 256, 0, s>>>(m, static_cast<float*>(out), ld_out, pieces, fast);
  else fp8_dequantize_kernel<__nv_bfloat16><<<static_cast<int>(blocks), 256, 0, s>>>(m, static_cast<__nv_bfloat16*>(out), ld_out, pieces, fast);
  check("fp8_dequantize");
}

}  // namespace himuon
