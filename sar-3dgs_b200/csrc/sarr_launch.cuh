// Launch helper of the multi-kernel operators (codebook, clipping): a launch
// that may start before its predecessor on the stream has finished
// (programmatic dependent launch).
#ifndef SARR_LAUNCH_CUH_
#define SARR_LAUNCH_CUH_

#include <cuda_runtime.h>
#include <stdint.h>

namespace sarr {

// Lets the next kernel of the stream that was launched as `dependent` place its
// CTAs. Its reads of this kernel's results still wait for this kernel's end.
__device__ __forceinline__ void dependents_may_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Waits for the end of the kernel before this one (returns at once in a launch
// that is not `dependent`). Every thread of a dependent kernel calls it before
// its first access to memory that an earlier kernel writes or reads.
__device__ __forceinline__ void wait_for_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

struct LaunchShape {
  dim3 grid;
  unsigned threads;
  size_t smem;
  bool dependent;  // may start before the previous kernel of the stream ends
};

template <typename... KArgs, typename... Args>
cudaError_t launch(void (*kernel)(KArgs...), const LaunchShape& shape, cudaStream_t stream,
                   Args&&... args) {
  if (!shape.dependent) {  // costs the host less than a launch with attributes
    kernel<<<shape.grid, shape.threads, shape.smem, stream>>>(static_cast<KArgs>(args)...);
    return cudaGetLastError();
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = shape.grid;
  cfg.blockDim = dim3(shape.threads);
  cfg.dynamicSmemBytes = shape.smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

}  // namespace sarr

#endif  // SARR_LAUNCH_CUH_
