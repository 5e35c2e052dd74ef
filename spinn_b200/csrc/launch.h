// launch.h -- launch helper of the decoder-serving operators.
#pragma once
#include "internal.h"

namespace spinn {

// Launches `kernel` as a programmatic dependent of the kernel queued before it on `st`: its
// launch overlaps that kernel's tail, and the kernel itself calls griddep_wait() before it reads
// anything.
template <typename... P, typename... A>
int launch_dependent(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  SPINN_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...));
  return 0;
}

}  // namespace spinn
