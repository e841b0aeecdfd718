// Kernels of one call that follow each other on a stream: the next one is
// launched while its predecessor still runs and waits, on the device, for the
// predecessor's memory -- the launch latency falls into the predecessor's time.
#pragma once

#include <cuda_runtime.h>

#include <utility>

namespace vg {

// In the predecessor: the successor may be launched once every CTA got here.
__device__ __forceinline__ void chain_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// In the successor, by every thread before anything that depends on the
// predecessor -- and before leaving: the kernel after the successor relies on
// the successor having waited.
__device__ __forceinline__ void chain_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Launches a kernel that begins with chain_wait behind one with chain_release.
template <class... Params, class... Args>
cudaError_t launch_chained(void (*kern)(Params...), dim3 grid, unsigned threads, size_t smem, cudaStream_t s,
                           Args &&...args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
}

}  // namespace vg
