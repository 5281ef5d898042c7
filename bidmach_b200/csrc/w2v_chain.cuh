// Kernels that follow one another on a stream, each launched before the one before it has ended: the
// launch and what a kernel does before it needs its inputs overlap the end of its predecessor.
#pragma once

#include <cuda_runtime.h>

#include <utility>

#include "w2v_internal.h"

namespace w2v {

// Every kernel that launch_chained starts calls this in all its threads before it touches global memory.
// What the kernels before it wrote is visible then.
__device__ __forceinline__ void chain_wait() {
  asm volatile("griddepcontrol.launch_dependents;\n\tgriddepcontrol.wait;" ::: "memory");
}

template <typename... P, typename... A>
int launch_chained(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t s, A &&...args) {
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t c = {};
  c.gridDim = grid;
  c.blockDim = dim3(threads);
  c.dynamicSmemBytes = smem;
  c.stream = s;
  c.attrs = &attr;
  c.numAttrs = 1;
  count_launch(1);
  return (int)cudaLaunchKernelEx(&c, kernel, P(std::forward<A>(args))...);
}

}  // namespace w2v
