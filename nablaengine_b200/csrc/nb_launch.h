// Launches that overlap with the kernel before them.
#pragma once
#include <cuda_runtime.h>

namespace nbtrain {

// Launch a kernel that may start while the one before it in the stream ends: it has to wait for it
// (griddepcontrol.wait) before its first access to memory that the other writes or still reads.
template <class... P, class... A>
int launch_after(cudaStream_t stream, int blocks, int threads, size_t smem, void (*kernel)(P...), A... args) {
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(blocks);
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  config.attrs = &attr;
  config.numAttrs = 1;
  return (int)cudaLaunchKernelEx(&config, kernel, static_cast<P>(args)...);
}

}  // namespace nbtrain
