// launch.h - launches that overlap the end of the kernel before them.
//
// A kernel launched here may start while its predecessor in the stream still
// runs: it sets itself up and then waits (wait_for_predecessor) until that grid
// has ended and its writes are visible, before it touches global memory.  Each
// kernel lets its successor do the same from its own start on
// (let_successor_start), so a chain of short kernels pays the launch latency
// once.  Behind any other kernel or operation the launch is an ordinary one.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>

namespace rab {

#ifdef __CUDACC__
__device__ __forceinline__ void wait_for_predecessor() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ void let_successor_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
#endif

// `args`: pointers to the kernel's parameters, of exactly its parameter types
template <typename... Params>
int launch_overlapped(void (*kernel)(Params...), dim3 grid, unsigned threads, size_t smem,
                      cudaStream_t stream, const Params*... args) {
  cudaLaunchAttribute overlap;
  overlap.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  overlap.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = &overlap;
  cfg.numAttrs = 1;
  void* list[] = {const_cast<void*>(static_cast<const void*>(args))...};
  return static_cast<int>(
      cudaLaunchKernelExC(&cfg, reinterpret_cast<const void*>(kernel), list));
}

}  // namespace rab
