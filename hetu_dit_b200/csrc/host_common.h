// Host-side helpers shared by the C-ABI translation units: thread-local error
// text, CUDA error mapping, and the per-device status block that kernels write
// to when one of their bounded waits runs out.
#pragma once
#include <cuda_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/hdit.h"

namespace hdit {

// printf-style; stores the text for hdit_last_error() and returns `code`.
int set_error(int code, const char* fmt, ...);

// Device pointer (valid on the current device) of the int32[16] status block.
// Lazily created; returns nullptr and sets the error text on failure.
int32_t* device_status_ptr();

#define HDIT_CUDA_OK(expr)                                                                       \
  do {                                                                                           \
    cudaError_t _e = (expr);                                                                     \
    if (_e != cudaSuccess)                                                                       \
      return ::hdit::set_error(HDIT_ERR_CUDA, "%s failed: %s (%s:%d)", #expr, cudaGetErrorString(_e), \
                               __FILE__, __LINE__);                                              \
  } while (0)

// Launch in stream order, but let the grid start while the kernel before it in the stream drains: its CTAs are
// scheduled, set up their barriers and tensor memory and then stand in grid_dependency_wait() until that kernel has
// completed and its writes are visible. Every kernel launched this way calls grid_dependency_wait() in all threads before
// its first access to global memory, and grid_dependency_release() so that the kernel after it may do the same. What the
// kernel before it writes changes while this kernel already runs, so none of them reads activations by the read-only path
// (__ldg(), const __restrict__ parameters), which promises data that is constant for the kernel's lifetime. Parameters of a
// layer may be read by it: copy_pieces_kernel, the one kernel here that writes them, lets the next one start only when it
// has finished.
// Measured: PipeFusion patch (scatter + attention) 127.7 -> 119.5 us, SD3-shaped step 20.8 -> 20.3 ms, SD3-shaped request
// 42.0 -> 41.3 ms, a 453 MB re-slice 74.3 -> 72.1 us a call.
template <typename... KernelArgs, typename... Args>
cudaError_t launch_overlapped(void (*kernel)(KernelArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                              unsigned cluster, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, static_cast<Args&&>(args)...);
  if (err != cudaSuccess) (void)cudaGetLastError();  // reported here, not once more by whoever launches next
  return err;
}

// Lets a kernel be launched with up to kBytes of dynamic shared memory. The limit belongs to the kernel on its device, not to a
// call or a host thread: every call sets the same one, the most that any call takes, so that none lowers it between another
// thread's set-up and launch.
template <auto kKernel, int kBytes>
cudaError_t allow_shared_memory() {
  static thread_local int last_dev = -1;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || dev == last_dev) return e;
  e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
  if (e == cudaSuccess) last_dev = dev;
  return e;
}

__device__ __forceinline__ void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_dependency_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Device-side: record the first failure of this launch and raise the CTA abort flag.
__device__ __forceinline__ void report_failure(int32_t* status, volatile int* abort_flag, int code, int where,
                                               int iter) {
  *abort_flag = 1;
  if (status != nullptr && atomicCAS(status, 0, code) == 0) {
    status[1] = static_cast<int32_t>(blockIdx.x);
    status[2] = where;
    status[3] = iter;
    __threadfence_system();
  }
}

}  // namespace hdit
