// tg_launch.cuh -- host-side launch helpers of the paged-cache kernels.
#pragma once

#include <cuda_runtime.h>

#include <mutex>
#include <utility>

namespace tg {

// A launch that may start while the kernel before it on the stream runs (its
// griddep_wait orders the memory).
template <typename... KArgs, typename... Args>
cudaError_t launch_chained(void (*fn)(KArgs...), dim3 grid, dim3 block, size_t smem,
                           cudaStream_t st, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, fn, std::forward<Args>(args)...);
}

// Raises a kernel's dynamic shared-memory limit to the most a CTA can have,
// once per device; `done` [64] is the kernel's own.  Contexts of several
// threads may come here at once.
template <typename F>
cudaError_t allow_max_smem(F* fn, bool* done) {
  static std::mutex mu;
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  std::lock_guard<std::mutex> lock(mu);
  if (done[dev]) return cudaSuccess;
  cudaError_t e =
      cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
  if (e == cudaSuccess) done[dev] = true;
  return e;
}

}  // namespace tg
