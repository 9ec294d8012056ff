// Launches that report their own result.  The runtime also keeps the error of
// a failed call as the "last" one: a launch that asked for the last error would
// report what an earlier call left behind, and one that left its own there
// would fail a later, healthy call.
#pragma once
#include <cuda_runtime.h>

#include "../../include/taccel_b200.h"

namespace tac {

inline int status(cudaError_t e) {
  if (e == cudaSuccess) return TAC_OK;
  cudaGetLastError();
  return TAC_E_CUDA;
}

template <typename... P, typename... A>
int launch(void (*kernel)(P...), unsigned grid, int threads, size_t smem, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  return status(cudaLaunchKernelEx(&cfg, kernel, P(args)...));
}

}  // namespace tac
