// Launch helpers of the kernels that are chained on a stream: programmatic dependent launch, overlap checks.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "../core/common.h"

namespace tvb {

// Queues `kernel` so that it may begin while the previous kernel of the stream ends (its CTAs take SMs as they come free).
// The kernel executes griddepcontrol.wait in every CTA before it touches global memory, so nothing it reads or writes is
// early; what overlaps is the launch itself and whatever set-up the kernel does before that wait. cluster: CTAs per cluster.
template <class... Params, class... Args>
int launch_dependent(const char* name, void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  TVB_CUDA(cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...));
  return launched(name, grid, block, smem, stream);
}

template <class... Params, class... Args>
int launch_dependent_cluster(const char* name, void (*kernel)(Params...), int cluster, dim3 grid, dim3 block, size_t smem,
                             cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  TVB_CUDA(cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...));
  return launched(name, grid, block, smem, stream);
}

// Whether two ranges of memory share a byte (an empty or NULL range shares none).
inline bool overlap(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
  if (a == nullptr || b == nullptr || a_bytes <= 0 || b_bytes <= 0) return false;
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + static_cast<uintptr_t>(b_bytes) && y < x + static_cast<uintptr_t>(a_bytes);
}

}  // namespace tvb
