// Product of two 8-bit matrices with a scale for each block of 128:  c_ij = sum over blocks b of  sa_i,b * sb_j,b * (sum of the block's qa_ik qb_jk).
//
// The tensor core sums the 128 products of a block in fp32; the blocks are added up outside of it, because every block has scales of its own:
// c is in registers, and each block's sums are read from tensor memory, scaled and added there in fp32.  As b has blocks of 128 rows, a thread, which has
// one row of a and 128 columns, needs one factor a block.
//
// A CTA pair has 256 x 256 of c (gemm2_sm100.cu has the protocol of pairs): a block of 256 x 256 x 128 takes its tensor cores 512 cycles, in which each CTA
// loads 32 KB and its eight summing warps read 128 KB of tensor memory and do 128 multiply-adds of two values a thread.  With one CTA to a tile of 128 x 256
// it would be 48 KB to load in the same time, more than an SM takes in.  Two accumulators, so that one block is added up beside the products of the next.
#include "fp8.h"
#include "gemm_epilogue.cuh"
#include "himuon.h"
#include "pair_common.cuh"
#include "sm100_common.cuh"
#include "tma_host.h"

#include <atomic>

namespace himuon {

namespace {

constexpr int F8_THREADS = 384;      // warps 0-3: TMA, MMA, none, none; 4-11: sums, two groups of four
// Registers of a thread at launch, and after the first four warps have given some to the others, whose sums take 128.
constexpr int F8_REGS = 168, F8_REGS_FEW = 104, F8_REGS_SUMS = 200;
static_assert(F8_REGS_FEW + 2 * F8_REGS_SUMS <= 3 * F8_REGS, "more registers than the block was launched with");
constexpr int F8_STAGES = 6;
constexpr int F8_K = 128;            // values of a block, a 128-byte row of shared memory
constexpr uint32_t F8_A = BM * F8_K, F8_STAGE = 2 * F8_A;

struct Fp8Dev {
  const float *sa, *sb;
  void* c;
  long long sa_row, sa_col, sb_row, sb_col;
  int a_block;                       // rows of a block of a
  int rows, cols, tiles_m, tiles_n, kblocks;
  int* status;
};

__device__ __forceinline__ void umma2_f8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate, uint32_t e) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(e)
      : "memory");
}
// fp32 sums of e4m3 values (format 0), both operands along K.
constexpr uint32_t idesc_e4m3(int m, int n) { return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24); }

}  // namespace

template <bool F32>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(F8_THREADS, 1)
fp8_product_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmC, Fp8Dev p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_up_1024(smem_raw);
  uint8_t* slabs = smem + F8_STAGES * F8_STAGE;
  uint64_t* full = reinterpret_cast<uint64_t*>(slabs + 2 * SLAB_BYTES);
  uint64_t* empty = full + F8_STAGES;
  uint64_t* tfull = empty + F8_STAGES;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = warp_id(), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < F8_STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(&tfull[a], 1); mbar_init(&tempty[a], 16); }     // eight summing warps in each CTA
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) tmem_alloc2(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                // the peer's barriers exist before anything signals them
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  const int first = blockIdx.x >> 1, n_pairs = gridDim.x >> 1, total = p.tiles_m * p.tiles_n;

  if (warp < 4) {
  registers_down<F8_REGS_FEW>();
  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer (both CTAs)
    const uint32_t e = elect_one();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int tile = first; ok && tile < total; tile += n_pairs) {
      const int nt = tile / p.tiles_m, m0 = (tile - nt * p.tiles_m) * 256 + static_cast<int>(rank) * BM, n0 = nt * 256 + static_cast<int>(rank) * BM;
      for (int kb = 0; kb < p.kblocks; ++kb) {
        if (!mbar_wait_warp(&empty[stage], phase ^ 1, abort_flag, p.status, 1)) { ok = false; break; }
        uint8_t* sA = smem + stage * F8_STAGE;
        mbar_expect_tx(&full[stage], 2 * F8_STAGE, leader ? e : 0);
        tma2_load_3d(sA, &tmA, &full[stage], kb * F8_K, m0, 0, e);
        tma2_load_3d(sA + F8_A, &tmB, &full[stage], kb * F8_K, n0, 0, e);
        if (++stage == F8_STAGES) { stage = 0; phase ^= 1; }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (leader CTA only)
    if (leader) {
      const uint32_t e = elect_one();
      constexpr uint32_t idesc = idesc_e4m3(256, 256);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int tile = first; ok && tile < total; tile += n_pairs) {
        for (int kb = 0; kb < p.kblocks; ++kb) {
          if (!mbar_wait_warp(&tempty[acc], acc_phase ^ 1, abort_flag, p.status, 2) || !mbar_wait_warp(&full[stage], phase, abort_flag, p.status, 2)) { ok = false; break; }
          tc_fence_after();
          const uint32_t a_base = smem_u32(smem + stage * F8_STAGE);
          const uint64_t a_desc = umma_smem_desc(a_base, 16, 1024), b_desc = umma_smem_desc(a_base + F8_A, 16, 1024);
#pragma unroll
          for (int k = 0; k < 4; ++k)                // 32 values an instruction
            umma2_f8(tmem_base + static_cast<uint32_t>(acc * 256), desc_at(a_desc, k * 32), desc_at(b_desc, k * 32), idesc, k > 0 ? 1u : 0u, e);
          const uint32_t e_addr = smem_u32(&empty[stage]), f_addr = smem_u32(&tfull[acc]);
          umma2_commit(f_addr, e);
          umma2_commit(map_to_cta(f_addr, 1), e);
          umma2_commit(e_addr, e);                   // this CTA's producer
          umma2_commit(map_to_cta(e_addr, 1), e);    // the peer's producer
          if (++stage == F8_STAGES) { stage = 0; phase ^= 1; }
          acc ^= 1;
          if (acc == 0) acc_phase ^= 1;
        }
      }
    }
  }
  } else {
    registers_up<F8_REGS_SUMS>();
    // ------------------------------------------------------------ sums (both CTAs, own 128 rows of the tile, one a thread; 128 columns a group)
    const int ew = warp & 3, group = (warp - 4) >> 2, row_in_tile = ew * 32 + lane;
    const uint32_t tempty_lead = map_to_cta(smem_u32(tempty), 0);
    const bool issuer = ew == 0 && lane == 0;
    uint8_t* slab = slabs + group * SLAB_BYTES;
    uint8_t* my_row = slab + row_in_tile * 128;
    const uint32_t t_group = tmem_base + (static_cast<uint32_t>(ew * 32) << 16) + static_cast<uint32_t>(group * 128);
    if (issuer) tma_prefetch_desc(&tmC);
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int tile = first; ok && tile < total; tile += n_pairs) {
      const int nt = tile / p.tiles_m, m0 = (tile - nt * p.tiles_m) * 256 + static_cast<int>(rank) * BM, n0 = nt * 256 + group * 128;
      const int row = m0 + row_in_tile;
      const bool mine = row < p.rows && n0 < p.cols;           // (else there is nothing to scale: zeros)
      const float* sa = p.sa + static_cast<long long>(mine ? row / p.a_block : 0) * p.sa_row;
      const float* sb = p.sb + static_cast<long long>(mine ? n0 / 128 : 0) * p.sb_row;
      float next = mine ? sa[0] * sb[0] : 0.f;
      f32x2 c[64];
#pragma unroll
      for (int j = 0; j < 64; ++j) c[j] = pack2(0.f, 0.f);
#pragma unroll 1
      for (int kb = 0; kb < p.kblocks; ++kb) {
        const f32x2 scale = pack2(next, next);
        if (mine && kb + 1 < p.kblocks) next = sa[(kb + 1) * p.sa_col] * sb[(kb + 1) * p.sb_col];
        ok = mbar_wait(&tfull[acc], acc_phase, abort_flag, p.status, 3);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        tc_fence_after();
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          uint32_t v[16];
          tmem_ld16(t_group + static_cast<uint32_t>(acc * 256) + q * 16, v);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 8; ++j) c[q * 8 + j] = fma2(pack2(v[2 * j], v[2 * j + 1]), scale, c[q * 8 + j]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_remote(tempty_lead + acc * 8);
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
      }
      // the 128 threads of a group meet on named barriers below, so they also leave together when a wait runs out
      ok = named_barrier_and(1 + 2 * group, 128, ok);
      if (!ok) break;
      if (m0 >= p.rows) continue;                              // uniform
#pragma unroll
      for (int sl = 0; sl < (F32 ? 4 : 2); ++sl) {             // slabs of 32 or 64 columns
        const int col = n0 + sl * (F32 ? 32 : 64);
        if (col >= p.cols) break;
        if (issuer) tma_store_wait_read<0>();
        named_barrier(1 + 2 * group, 128);                     // the slab is free
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint4 o;
          if constexpr (F32) {
            float f[4];
            unpack2(c[sl * 16 + 2 * j], f[0], f[1]);
            unpack2(c[sl * 16 + 2 * j + 1], f[2], f[3]);
            o = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
          } else {
            uint32_t w[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              float lo, hi;
              unpack2(c[sl * 32 + 4 * j + t], lo, hi);
              w[t] = pack_bf16x2(lo, hi);
            }
            o = make_uint4(w[0], w[1], w[2], w[3]);
          }
          *reinterpret_cast<uint4*>(my_row + ((j ^ (row_in_tile & 7)) << 4)) = o;
        }
        fence_proxy_async_smem();
        named_barrier(2 + 2 * group, 128);                     // the slab is complete
        if (issuer) {
          tma_store_3d(&tmC, slab, col, m0, 0);
          tma_store_commit();
        }
      }
    }
    if (issuer) tma_store_wait_all();
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                  // neither CTA leaves while the other may still signal or read it
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc2(tmem_base, 512);
  }
}

static CUtensorMap bytes_map(const Fp8Matrix& m) {
  const uint64_t dims[3] = {static_cast<uint64_t>(m.cols), static_cast<uint64_t>(m.rows), 1};
  const uint64_t strides[2] = {static_cast<uint64_t>(m.ld), static_cast<uint64_t>(m.ld) * static_cast<uint64_t>(m.rows)};
  const uint32_t box[3] = {F8_K, BM, 1};
  return make_tmap(m.values, 3, dims, strides, box, 1, true);
}

// CTA pairs that can be resident at once on the current device.  (Callers and the autograd engine's threads may ask at the same time.)
template <class Kernel>
static int pairs_at_once(Kernel kernel, size_t smem) {
  static std::atomic<int> most[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  const bool known = dev >= 0 && dev < 64;
  int n = known ? most[dev].load(std::memory_order_relaxed) : 0;
  if (n == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(num_sms());
    cfg.blockDim = dim3(F8_THREADS);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 2; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) {
      cudaGetLastError();
      n = num_sms() / 2;
    }
    if (known) most[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

void fp8_product(const Fp8Matrix& a, const Fp8Matrix& b, void* c, long long ld_c, int out_fp32, cudaStream_t s) {
  constexpr size_t SMEM = 1024 + F8_STAGES * F8_STAGE + 2 * SLAB_BYTES + 256;
  static_assert(SMEM <= 232448, "shared memory budget of one CTA exceeded");
  const int esz = out_fp32 ? 4 : 2;
  const auto kernel = out_fp32 ? fp8_product_kernel<true> : fp8_product_kernel<false>;
  if (a.rows <= 0 || b.rows <= 0 || a.cols <= 0 || a.cols != b.cols || b.block_rows != 128 || ld_c < b.rows || ld_c * esz % 16)
    throw std::runtime_error("himuon fp8_product: bad sizes");
  const cudaError_t set = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(SMEM));
  if (set != cudaSuccess) throw std::runtime_error(std::string("himuon fp8_product: ") + cudaGetErrorString(set));
  Fp8Dev p{};
  p.sa = a.scales; p.sb = b.scales; p.c = c;
  p.sa_row = a.scale_row; p.sa_col = a.scale_col; p.sb_row = b.scale_row; p.sb_col = b.scale_col;
  p.a_block = a.block_rows;
  p.rows = a.rows; p.cols = b.rows;
  p.tiles_m = (a.rows + 255) / 256;
  p.tiles_n = (b.rows + 255) / 256;
  p.kblocks = (a.cols + F8_K - 1) / F8_K;
  p.status = status_word_ptr();
  const long long total = static_cast<long long>(p.tiles_m) * p.tiles_n;
  if (total >= (1LL << 30)) throw std::runtime_error("himuon fp8_product: too many tiles for one launch");
  const uint64_t dims[3] = {static_cast<uint64_t>(b.rows), static_cast<uint64_t>(a.rows), 1};
  const uint64_t strides[2] = {static_cast<uint64_t>(ld_c) * esz, static_cast<uint64_t>(ld_c) * esz * dims[1]};
  const uint32_t box[3] = {static_cast<uint32_t>(128 / esz), BM, 1};
  const CUtensorMap tc = make_tmap(c, 3, dims, strides, box, esz, true);
  const int pairs = pairs_at_once(kernel, SMEM);
  kernel<<<2 * static_cast<int>(total < pairs ? total : pairs), F8_THREADS, SMEM, s>>>(bytes_map(a), bytes_map(b), tc, p);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) throw std::runtime_error(std::string("himuon fp8_product launch failed: ") + cudaGetErrorString(e));
}

}  // namespace himuon
