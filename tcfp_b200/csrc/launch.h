// Host-side plumbing shared by the translation units of libtcfp_b200:
// thread-local error text, CUDA error mapping, device properties.
#pragma once

#include <cuda_runtime.h>
#include <stdarg.h>
#include <stdint.h>

#include "../../include/tcfp_b200.h"

namespace tcfp {

// records a printf-style message for tcfp_last_error() and returns `code`
int fail(int code, const char* fmt, ...);
// number of SMs of the current device (cached per device)
int sm_count();
// SMs the persistent GEMM grids may occupy: sm_count() minus the calling thread's
// tcfp_set_sm_reserve() (SMs left free for a collective running beside the GEMM)
int gemm_sm_budget();

// Launch that may begin while the kernel before it in the stream is still finishing (programmatic dependent launch): the
// kernel must call wait_for_stream() before it touches global memory.  cfg.attrs has room for one more attribute behind
// numAttrs.
inline void allow_early_start(cudaLaunchConfig_t& cfg) {
  cudaLaunchAttribute& a = cfg.attrs[cfg.numAttrs++];
  a.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  a.val.programmaticStreamSerializationAllowed = 1;
}

template <typename... Params, typename... Args>
cudaError_t launch_early(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args... args) {
  cudaLaunchAttribute attrs[1];
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attrs;
  allow_early_start(cfg);
  return cudaLaunchKernelEx(&cfg, kernel, Params(args)...);
}

#ifdef __CUDACC__
// The other half: lets the next kernel's blocks take their places as soon as every block of this one has started, then
// waits until the kernel before this one is done and its writes are visible.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_stream() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
#endif

}  // namespace tcfp

#define CUDA_TRY(expr)                                                                         \
  do {                                                                                         \
    cudaError_t _e = (expr);                                                                   \
    if (_e != cudaSuccess)                                                                     \
      return ::tcfp::fail(TCFP_ERR_CUDA, "%s failed: %s", #expr, cudaGetErrorString(_e));      \
  } while (0)
