// Attributes of a kernel, set once on each device it is launched on (they belong to the
// device, not to the process).
#pragma once
#include <cuda_runtime_api.h>

#include <atomic>
#include <cstdint>

namespace tlx {

// Shared memory opt-in of `kernel`, and the carveout for all the CTAs an SM is to hold.
// `done`: a bit for each device; a device past 63 is set up at every call.
inline bool setup_kernel(const void* kernel, int smem, std::atomic<uint64_t>& done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0) return false;
  const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
      cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared) !=
          cudaSuccess)
    return false;
  done.fetch_or(bit, std::memory_order_relaxed);
  return true;
}

}  // namespace tlx
