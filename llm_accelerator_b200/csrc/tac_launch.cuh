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

// The same for a kernel whose threads all begin with after_previous(): its CTAs
// may take their places while the last ones of the kernel before it run, if
// that one lets them (let_next), which spares the gap between two launches.
template <typename... P, typename... A>
int launch_behind(void (*kernel)(P...), unsigned grid, int threads, size_t smem, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return status(cudaLaunchKernelEx(&cfg, kernel, P(args)...));
}

// All kernels before this one have completed, and their results are visible.
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;\n" ::: "memory"); }
// The next kernel's CTAs may start where there is room; called by every CTA.
__device__ __forceinline__ void let_next() { asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory"); }

}  // namespace tac
