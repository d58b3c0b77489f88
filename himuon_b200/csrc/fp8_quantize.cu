// Matrices in 8 bits: e4m3 values and a power of two for each block of (1, 128) or (128, 128) of them.
//
//   scale = the least 2^k with max |x| <= 448 * 2^k (1 where the block holds nothing but zeros, 2^-110 at the least),  q = rn_e4m3(x / scale)
//
// A power of two makes the division exact, so that q has one rounding of x (2^-4 of it at most, or 2^-10 of the scale) and no value next to a tie
// hangs on the rounding of a quotient; it costs up to one bit of range at the lower end, of 17.  A value that is not finite becomes NaN and has no part
// in its block's scale.  Below 2^-110 * 2^-10 there is nothing left, also not what this build's arithmetic would flush.
//
// Bounded by memory: a block of 256 threads has 128 x 128 values, 8 x 8 a thread, reads them once and writes each wanted copy, as they lie
// and turned around (through shared memory), with the same scales' maxima from one pass.
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
__device__ __forceinline__ uint32_t finite_bits(float x) {
  const uint32_t b = __float_as_uint(x) & 0x7FFFFFFFu;
  return b < 0x7F800000u ? b : 0u;
}
__device__ __forceinline__ float nan_for_infinite(float x) {
  return (__float_as_uint(x) & 0x7FFFFFFFu) >= 0x7F800000u ? __uint_as_float(0x7FFFFFFFu) : x;
}
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

template <typename T>
__device__ __forceinline__ void load8(const T* p, int valid, bool whole, float (&f)[8]) {
  if (whole) {
    if constexpr (sizeof(T) == 2) {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) { f[2 * j] = bf16_lo(w[j]); f[2 * j + 1] = bf16_hi(w[j]); }
    } else {
      const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
      f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = j < valid ? as_float(p[j]) : 0.f;
  }
}

template <typename T>
__global__ void __launch_bounds__(256) fp8_quantize_kernel(Fp8QuantizeArgs a, int tiles_c, int aligned) {
  __shared__ uint32_t s_col[QT];
  __shared__ uint32_t s_all;
  __shared__ uint2 s_turned[QT * 16];                  // [column][group of 8 rows, swizzled]
  const int tr = threadIdx.x >> 4, tc = threadIdx.x & 15;
  const long long rblk = blockIdx.x / tiles_c, cblk = blockIdx.x - rblk * tiles_c;
  const long long r0 = rblk * QT + tr * 8, c0 = cblk * QT + tc * 8;
  const bool turn = a.turned.values != nullptr;
  float v[8][8];
  const int valid = static_cast<int>(a.cols - c0 < 8 ? a.cols - c0 : 8);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const bool in = r0 + i < a.rows;
    load8(reinterpret_cast<const T*>(a.x) + (r0 + i) * a.ld + c0, in ? valid : 0, in && valid == 8 && aligned, v[i]);
  }
  const bool whole_scale = (a.straight.values && a.straight.block_rows == QT) || (turn && a.turned.block_rows == QT);
  if (threadIdx.x < QT) s_col[threadIdx.x] = 0;
  if (threadIdx.x == 0) s_all = 0;
  __syncthreads();
  uint32_t row_max[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, finite_bits(v[i][j]));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    row_max[i] = m;
  }
  if (whole_scale) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, row_max[i]);
    if (tc == 0) atomicMax(&s_all, m);
  }
  if (turn && a.turned.block_rows == 1) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max(m, finite_bits(v[i][j]));
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 16));
      if ((threadIdx.x & 16) == 0) atomicMax(&s_col[tc * 8 + j], m);
    }
  }
  __syncthreads();
  const int all = whole_scale ? scale_exponent(s_all) : 0;
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) v[i][j] = nan_for_infinite(v[i][j]);

  if (a.straight.values) {
    const Fp8Out& o = a.straight;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int k = o.block_rows == QT ? all : scale_exponent(row_max[i]);
      const float by = power_of_two(-k);
      if (r0 + i < a.rows) {
        if (c0 < o.ld)                                 // (behind the last column, up to the row's end, are zeros)
          *reinterpret_cast<uint2*>(static_cast<uint8_t*>(o.values) + (r0 + i) * o.ld + c0) =
              make_uint2(pack4(v[i][0] * by, v[i][1] * by, v[i][2] * by, v[i][3] * by), pack4(v[i][4] * by, v[i][5] * by, v[i][6] * by, v[i][7] * by));
        if (tc == 0 && o.block_rows == 1) o.scales[(r0 + i) * o.scale_row + cblk * o.scale_col] = power_of_two(k);
      }
    }
    if (threadIdx.x == 0 && o.block_rows == QT) o.scales[rblk * o.scale_row + cblk * o.scale_col] = power_of_two(all);
  }
  if (turn) {
    const Fp8Out& o = a.turned;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = tc * 8 + j;
      const float by = power_of_two(-(o.block_rows == QT ? all : scale_exponent(s_col[c])));
      s_turned[c * 16 + (tr ^ tc)] =
          make_uint2(pack4(v[0][j] * by, v[1][j] * by, v[2][j] * by, v[3][j] * by), pack4(v[4][j] * by, v[5][j] * by, v[6][j] * by, v[7][j] * by));
    }
    if (o.block_rows == 1) {
      if (threadIdx.x < QT && cblk * QT + threadIdx.x < a.cols)
        o.scales[(cblk * QT + threadIdx.x) * o.scale_row + rblk * o.scale_col] = power_of_two(scale_exponent(s_col[threadIdx.x]));
    } else if (threadIdx.x == 0) {
      o.scales[cblk * o.scale_row + rblk * o.scale_col] = power_of_two(all);
    }
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

// Four values a thread and turn, so that 32 threads write 512 bytes in a row.
template <typename T>
__global__ void __launch_bounds__(256) fp8_dequantize_kernel(Fp8Matrix m, T* out, long long ld_out, int groups, int fast, long long total) {
  for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < total; i += static_cast<long long>(gridDim.x) * 256) {
    const long long row = i / groups;
    const int col = static_cast<int>(i - row * groups) * 4;
    const uint8_t* src = static_cast<const uint8_t*>(m.values) + row * m.ld + col;
    T* dst = out + row * ld_out + col;
    const float scale = m.scales[(m.block_rows == 1 ? row : row / QT) * m.scale_row + (col / QT) * m.scale_col];
    const int valid = m.cols - col < 4 ? m.cols - col : 4;
    uint32_t q = 0;
    if (fast) q = *reinterpret_cast<const uint32_t*>(src);
    else
      for (int j = 0; j < valid; ++j) q |= static_cast<uint32_t>(src[j]) << (8 * j);
    const float2 lo = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(q & 0xFFFFu), __NV_E4M3)));
    const float2 hi = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(q >> 16), __NV_E4M3)));
    const float f[4] = {lo.x * scale, lo.y * scale, hi.x * scale, hi.y * scale};
    if (fast) {
      if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(dst) = make_float4(f[0], f[1], f[2], f[3]);
      else *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < valid) put(dst + j, f[j]);
    }
  }
}

void check(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) throw std::runtime_error(std::string("himuon ") + what + " launch failed: " + cudaGetErrorString(e));
}

}  // namespace

void fp8_quantize(const Fp8QuantizeArgs& a, cudaStream_t s) {
  if (a.rows <= 0 || a.cols <= 0) return;
  for (const Fp8Out* o : {&a.straight, &a.turned})
    if (o->values && ((o->block_rows != 1 && o->block_rows != QT) || o->ld % 16 || reinterpret_cast<uintptr_t>(o->values) % 16))
      throw std::runtime_error("himuon fp8_quantize: blocks of 1 or 128 rows, rows of multiples of 16 bytes");
  const long long tiles_c = (a.cols + QT - 1) / QT, tiles = (a.rows + QT - 1) / QT * tiles_c;
  if (tiles >= (1LL << 31)) throw std::runtime_error("himuon fp8_quantize: matrix too large for one launch");
  const int aligned = reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && a.ld % (a.fp32 ? 4 : 8) == 0;
  if (a.fp32) fp8_quantize_kernel<float><<<static_cast<int>(tiles), 256, 0, s>>>(a, static_cast<int>(tiles_c), aligned);
  else fp8_quantize_kernel<__nv_bfloat16><<<static_cast<int>(tiles), 256, 0, s>>>(a, static_cast<int>(tiles_c), aligned);
  check("fp8_quantize");
}

void fp8_dequantize(const Fp8Matrix& m, void* out, long long ld_out, int out_fp32, cudaStream_t s) {
  if (m.rows <= 0 || m.cols <= 0) return;
  const int groups = (m.cols + 3) / 4;
  const int fast = m.cols % 4 == 0 && m.ld % 4 == 0 && reinterpret_cast<uintptr_t>(m.values) % 4 == 0 && ld_out % 4 == 0 &&
                   reinterpret_cast<uintptr_t>(out) % 16 == 0;
  const long long total = static_cast<long long>(m.rows) * groups, blocks = (total + 255) / 256, most = static_cast<long long>(num_sms()) * 32;
  const int grid = static_cast<int>(blocks < most ? blocks : most);
  if (out_fp32) fp8_dequantize_kernel<float><<<grid, 256, 0, s>>>(m, static_cast<float*>(out), ld_out, groups, fast, total);
  else fp8_dequantize_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(m, static_cast<__nv_bfloat16*>(out), ld_out, groups, fast, total);
  check("fp8_dequantize");
}

}  // namespace himuon
