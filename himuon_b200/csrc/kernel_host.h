// What a launch needs to know of its kernel on the current device, asked once for each kernel and device.  (A process may use several devices, and callers
// and the autograd engine's threads may launch at the same time: what is kept is atomic, and each device has its own.)
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <stdexcept>
#include <string>

#include "himuon.h"

namespace himuon {

// Lets a kernel have `bytes` of dynamic shared memory, which it has to be allowed on every device.
template <typename K>
void allow_smem(K kernel, size_t bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = dev >= 0 && dev < 64 ? 1ull << dev : 0;
  if (bit && (done.load(std::memory_order_relaxed) & bit)) return;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  if (e != cudaSuccess) throw std::runtime_error(std::string("himuon: shared memory of a kernel: ") + cudaGetErrorString(e));
  done.fetch_or(bit, std::memory_order_relaxed);
}

// CTA pairs of a kernel that can be resident at once (GPCs with an odd number of free SMs leave one SM unpaired).
template <typename K>
int pairs_at_once(K kernel, int threads, size_t smem, std::atomic<int> (&most)[64]) {
  int dev = 0;
  cudaGetDevice(&dev);
  const bool known = dev >= 0 && dev < 64;
  int n = known ? most[dev].load(std::memory_order_relaxed) : 0;
  if (n == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(num_sms());
    cfg.blockDim = dim3(threads);
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

}  // namespace himuon
