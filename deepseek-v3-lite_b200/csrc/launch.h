// Host-side launch helper shared by the paged-cache and beam-search kernels.
#pragma once
#include <cuda_runtime.h>

namespace dsv3 {

// Launch that may begin while its predecessor in the stream still runs; the
// kernel waits for it (griddepcontrol.wait) before it reads anything.
template <typename Kern, typename... Args>
inline cudaError_t launch_dependent(Kern kern, dim3 grid, int block, cudaStream_t st, Args... args) {
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(block);
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

}  // namespace dsv3
