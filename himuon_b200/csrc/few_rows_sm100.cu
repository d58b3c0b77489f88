// Products of a few rows (newest tokens) with a large weight, whose bytes are all that counts:  y = x W^T  in bf16, the same of two
// weights with the gated activation between them, and the same in 8 bits with a scale for each block of 128.
//
// Rows of W are streamed from memory straight into the registers that mma.sync takes them from: 16 rows of W are the A operand, up to 8 rows of x the
// B operand.  (tcgen05.mma takes its operands from shared memory and leaves its sums in tensor memory; both detours cost more here than the tensor core's rate
// gives, which is not needed: 16 x 8 x 16 products for every 512 bytes of weight.)  The sum over the inner dimension may take it in any order, as long
// as both operands use the same: so a thread loads 16 bytes that lie together, and gives them to two products.  Lane l has row l / 4 and bytes 16 (l % 4) of a
// step of 64 bytes, of W and of x alike.
//
// A block has 16 rows of W; its eight warps share the inner dimension, and a cluster of up to eight blocks again, where 16 rows a block would leave SMs
// idle.  The parts meet in shared memory, in one order, so that bits repeat, and a row's do not depend on how many rows come with it.
#include <cooperative_groups.h>

#include "activations.cuh"
#include "fp8.h"
#include "gated_mlp.h"
#include "himuon.h"
#include "sm100_common.cuh"

namespace himuon {

namespace cg = cooperative_groups;

namespace {

enum { PLAIN, GATED, EIGHT_BITS };

constexpr int FEW_WARPS = 8;

struct FewDev {
  const uint8_t *x, *w0, *w1;          // rows of bytes
  long long ld_x, ld_w0, ld_w1;
  const float *sx, *sw;                // EIGHT_BITS
  long long sx_row, sx_col, sw_row, sw_col;
  int x_block;
  void *y, *gu;                        // (rows, outer) in bf16 or fp32; GATED: g | u or null (gated_mlp.h)
  uint8_t* gu_low;
  int rows, outer, inner_bytes, out_fp32;
};

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_e4m3(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 stream16(const uint8_t* p, bool ok) {
  return ok ? __ldcs(reinterpret_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0);
}

// NT: groups of eight rows of x.  ACT: of GATED.
template <int KIND, int NT, int ACT>
__global__ void __launch_bounds__(FEW_WARPS * 32) few_rows_kernel(FewDev p) {
  constexpr int MATS = KIND == GATED ? 2 : 1;
  constexpr int NX = NT * 8;
  constexpr int UNROLL = NT >= 4 ? 2 : 4;              // steps of 64 bytes whose loads are under way together
  extern __shared__ float s_part[];                    // [warp][matrix][16][NX], then [matrix][16][NX] of the block
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
  const cg::cluster_group cluster = cg::this_cluster();
  const int S = static_cast<int>(cluster.num_blocks()), part = static_cast<int>(cluster.block_rank());
  const int f0 = static_cast<int>(blockIdx.x / S) * 16;
  // this warp's share of the inner dimension, in blocks of 128 values where they have scales of their own and steps else
  constexpr int UNIT = KIND == EIGHT_BITS ? 128 : 64;
  const int units = (p.inner_bytes + UNIT - 1) / UNIT, shares = S * FEW_WARPS, share = part * FEW_WARPS + warp;
  const int u0 = static_cast<int>(static_cast<long long>(units) * share / shares), u1 = static_cast<int>(static_cast<long long>(units) * (share + 1) / shares);
  const bool ok0 = f0 + r < p.outer, ok1 = f0 + r + 8 < p.outer;
  const uint8_t *wa[MATS], *wb[MATS];
  wa[0] = p.w0 + (ok0 ? f0 + r : 0) * p.ld_w0 + t * 16;
  wb[0] = p.w0 + (ok1 ? f0 + r + 8 : 0) * p.ld_w0 + t * 16;
  if constexpr (MATS == 2) {
    wa[1] = p.w1 + (ok0 ? f0 + r : 0) * p.ld_w1 + t * 16;
    wb[1] = p.w1 + (ok1 ? f0 + r + 8 : 0) * p.ld_w1 + t * 16;
  }
  float acc[MATS][NT][4] = {};
  if constexpr (KIND == EIGHT_BITS) {
    const float* sw = p.sw + static_cast<long long>(f0 / 128) * p.sw_row;
    for (int u = u0; u < u1; u += UNROLL / 2) {        // two steps a block
      uint4 va[UNROLL], vb[UNROLL];
#pragma unroll
      for (int i = 0; i < UNROLL; ++i) {
        const int at = u * 128 + i * 64;
        const bool in = u + i / 2 < u1 && at + t * 16 < p.inner_bytes;
        va[i] = stream16(wa[0] + at, in && ok0);
        vb[i] = stream16(wb[0] + at, in && ok1);
      }
#pragma unroll
      for (int b = 0; b < UNROLL / 2; ++b) {
        if (u + b >= u1) break;
        const float w_scale = sw[(u + b) * p.sw_col];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int row = n * 8 + r;
          float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 2 * b; i < 2 * b + 2; ++i) {
            const int at = u * 128 + i * 64 + t * 16;
            const uint4 x = row < p.rows && at < p.inner_bytes ? *reinterpret_cast<const uint4*>(p.x + row * p.ld_x + at) : make_uint4(0, 0, 0, 0);
            mma_e4m3(c, va[i].x, vb[i].x, va[i].y, vb[i].y, x.x, x.y);
            mma_e4m3(c, va[i].z, vb[i].z, va[i].w, vb[i].w, x.z, x.w);
          }
#pragma unroll
          for (int j = 0; j < 2; ++j) {                // columns 2t and 2t + 1 of the product are rows of x
            const int col = n * 8 + 2 * t + j;
            const float s = col < p.rows ? w_scale * p.sx[(col / p.x_block) * p.sx_row + (u + b) * p.sx_col] : 0.f;
            acc[0][n][j] = fmaf(c[j], s, acc[0][n][j]);
            acc[0][n][2 + j] = fmaf(c[2 + j], s, acc[0][n][2 + j]);
          }
        }
      }
    }
  } else {
    for (int u = u0; u < u1; u += UNROLL) {
      uint4 va[MATS][UNROLL], vb[MATS][UNROLL];
#pragma unroll
      for (int i = 0; i < UNROLL; ++i) {
        const int at = (u + i) * 64;
        const bool in = u + i < u1 && at + t * 16 < p.inner_bytes;
#pragma unroll
        for (int m = 0; m < MATS; ++m) {
          va[m][i] = stream16(wa[m] + at, in && ok0);
          vb[m][i] = stream16(wb[m] + at, in && ok1);
        }
      }
#pragma unroll
      for (int i = 0; i < UNROLL; ++i) {
        if (u + i >= u1) break;
        const int at = (u + i) * 64 + t * 16;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int row = n * 8 + r;
          const uint4 x = row < p.rows && at < p.inner_bytes ? *reinterpret_cast<const uint4*>(p.x + row * p.ld_x + at) : make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int m = 0; m < MATS; ++m) {
            mma_bf16(acc[m][n], va[m][i].x, vb[m][i].x, va[m][i].y, vb[m][i].y, x.x, x.y);
            mma_bf16(acc[m][n], va[m][i].z, vb[m][i].z, va[m][i].w, vb[m][i].w, x.z, x.w);
          }
        }
      }
    }
  }
  // the warps' parts: row r (and r + 8) of W, rows 2t and 2t + 1 of each group of x
#pragma unroll
  for (int m = 0; m < MATS; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float* dst = s_part + ((warp * MATS + m) * 16 + r) * NX + n * 8 + 2 * t;
      dst[0] = acc[m][n][0];
      dst[1] = acc[m][n][1];
      dst[8 * NX] = acc[m][n][2];
      dst[8 * NX + 1] = acc[m][n][3];
    }
  __syncthreads();
  constexpr int VALUES = MATS * 16 * NX;
  float* s_sum = s_part + FEW_WARPS * VALUES;
  for (int i = threadIdx.x; i < VALUES; i += FEW_WARPS * 32) {
    float v = s_part[i];
#pragma unroll
    for (int w = 1; w < FEW_WARPS; ++w) v += s_part[w * VALUES + i];
    s_sum[i] = v;
  }
  if (S > 1) cluster.sync();
  else __syncthreads();
  // the blocks' parts: each block has its share of the values, neighbouring features next to one another
  constexpr int OUT = 16 * NX;
  const int o0 = OUT * part / S, o1 = OUT * (part + 1) / S;
  for (int o = o0 + threadIdx.x; o < o1; o += FEW_WARPS * 32) {
    const int f = o & 15, row = o >> 4;
    float v[MATS];
#pragma unroll
    for (int m = 0; m < MATS; ++m) {
      const int at = (m * 16 + f) * NX + row;
      v[m] = 0.f;
      for (int k = 0; k < S; ++k) v[m] += S > 1 ? cluster.map_shared_rank(s_sum, k)[at] : s_sum[at];
    }
    if (row < p.rows && f0 + f < p.outer) {
      const long long at = static_cast<long long>(row) * p.outer + f0 + f;
      if constexpr (KIND == GATED) {
        reinterpret_cast<__nv_bfloat16*>(p.y)[at] = __float2bfloat16_rn(activate<ACT>(v[0]) * v[1]);
        if (p.gu) {
          uint16_t* gu = static_cast<uint16_t*>(p.gu) + 2LL * row * p.outer + f0 + f;
          uint8_t* low = p.gu_low + 2LL * row * gated_low(p.outer) + f0 + f;
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            gu[m * p.outer] = static_cast<uint16_t>(__float_as_uint(v[m]) >> 16);
            low[m * gated_low(p.outer)] = static_cast<uint8_t>(__float_as_uint(v[m]) >> 8);
          }
        }
      } else if (p.out_fp32) {
        reinterpret_cast<float*>(p.y)[at] = v[0];
      } else {
        reinterpret_cast<__nv_bfloat16*>(p.y)[at] = __float2bfloat16_rn(v[0]);
      }
    }
  }
  if (S > 1) cluster.sync();                           // no block leaves while another may still read its sums
}

template <int KIND, int NT, int ACT>
void launch(const FewDev& p, cudaStream_t s) {
  constexpr size_t SMEM = sizeof(float) * (FEW_WARPS + 1) * (KIND == GATED ? 2 : 1) * 16 * NT * 8;
  const auto kernel = few_rows_kernel<KIND, NT, ACT>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(SMEM));
  if (e == cudaSuccess) {
    const int groups = (p.outer + 15) / 16, steps = (p.inner_bytes + 63) / 64;
    int S = 1;                                         // blocks that share a group's inner dimension: about four a SM, of two steps a warp or more
    while (S < 8 && groups * S < 3 * num_sms() && steps >= 2 * S * FEW_WARPS * 2) S *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(groups * S);
    cfg.blockDim = dim3(FEW_WARPS * 32);
    cfg.dynamicSmemBytes = SMEM;
    cfg.stream = s;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = S; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kernel, p);
  }
  if (e != cudaSuccess) throw std::runtime_error(std::string("himuon product of few rows: launch failed: ") + cudaGetErrorString(e));
}
template <int KIND, int ACT = 0>
void launch_rows(const FewDev& p, cudaStream_t s) {
  if (p.rows <= 0 || p.rows > kFewProductRows || p.outer <= 0 || p.inner_bytes <= 0 || p.inner_bytes % 16) throw std::runtime_error("himuon product of few rows: bad sizes");
  if (p.rows <= 8) launch<KIND, 1, ACT>(p, s);
  else if (p.rows <= 16) launch<KIND, 2, ACT>(p, s);
  else if (p.rows <= 32) launch<KIND, 4, ACT>(p, s);
  else launch<KIND, 8, ACT>(p, s);
}

}  // namespace

void few_rows_product(const void* x, long long ld_x, const void* w, long long ld_w, void* y, int rows, int inner, int outer, cudaStream_t s) {
  FewDev p{};
  p.x = static_cast<const uint8_t*>(x); p.ld_x = 2 * ld_x;
  p.w0 = static_cast<const uint8_t*>(w); p.ld_w0 = 2 * ld_w;
  p.y = y;
  p.rows = rows; p.outer = outer; p.inner_bytes = 2 * inner;
  launch_rows<PLAIN>(p, s);
}

void few_rows_gated_up(const GatedUpArgs& a, cudaStream_t s) {
  FewDev p{};
  p.x = static_cast<const uint8_t*>(a.x); p.ld_x = 2 * a.ld_x;
  p.w0 = static_cast<const uint8_t*>(a.wg); p.ld_w0 = 2 * a.ld_wg;
  p.w1 = static_cast<const uint8_t*>(a.wu); p.ld_w1 = 2 * a.ld_wu;
  p.y = a.h; p.gu = a.gu; p.gu_low = static_cast<uint8_t*>(a.gu_low);
  p.rows = a.rows; p.outer = a.inter; p.inner_bytes = 2 * a.hidden;
  switch (a.activation) {
    case kSilu: return launch_rows<GATED, kSilu>(p, s);
    case kGelu: return launch_rows<GATED, kGelu>(p, s);
    case kGeluTanh: return launch_rows<GATED, kGeluTanh>(p, s);
    case kRelu: return launch_rows<GATED, kRelu>(p, s);
  }
  throw std::runtime_error("himuon gated_mlp: unknown activation");
}

void few_rows_fp8_product(const Fp8Matrix& a, const Fp8Matrix& b, void* c, int out_fp32, cudaStream_t s) {
  if (a.cols != b.cols || b.block_rows != 128) throw std::runtime_error("himuon fp8_product: bad sizes");
  FewDev p{};
  p.x = static_cast<const uint8_t*>(a.values); p.ld_x = a.ld;
  p.w0 = static_cast<const uint8_t*>(b.values); p.ld_w0 = b.ld;
  p.sx = a.scales; p.sx_row = a.scale_row; p.sx_col = a.scale_col; p.x_block = a.block_rows;
  p.sw = b.scales; p.sw_row = b.scale_row; p.sw_col = b.scale_col;
  p.y = c; p.out_fp32 = out_fp32;
  p.rows = a.rows; p.outer = b.rows; p.inner_bytes = a.cols;
  launch_rows<EIGHT_BITS>(p, s);
}

}  // namespace himuon
