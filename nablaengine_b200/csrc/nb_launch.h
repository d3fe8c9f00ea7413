// Launches that overlap with the kernel before them.
#pragma once
#include <cuda_runtime.h>

namespace nbtrain {

struct Launch {
  cudaStream_t stream;
  int blocks, threads, smem = 0, cluster = 1;
};

// Launch a kernel that may start while the one before it in the stream ends: it has to wait for it (wait_for_last)
// before its first access to memory.
template <class... P, class... A> int launch_after(const Launch& l, void (*kernel)(P...), A... args) {
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)l.cluster, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(l.blocks);
  config.blockDim = dim3(l.threads);
  config.dynamicSmemBytes = (size_t)l.smem;
  config.stream = l.stream;
  config.attrs = attr;
  config.numAttrs = l.cluster > 1 ? 2 : 1;
  return (int)cudaLaunchKernelEx(&config, kernel, static_cast<P>(args)...);
}

}  // namespace nbtrain
