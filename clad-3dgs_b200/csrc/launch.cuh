// Launches that overlap the end of the kernel before them in the stream.
//
// A kernel launched by `launch_after` may start while its predecessor's last
// blocks run (programmatic dependent launch): its blocks get their places and
// then wait in `wait_before`, the first statement of every such kernel, until
// the predecessor is complete and its writes are visible. Every thread of every
// block passes it, so a kernel's end means that all kernels before it have
// ended too, and memory may be reused along the stream as usual. Behind
// anything but a kernel of this kind the launch is an ordinary one.
//
// Such a kernel's pointers to what earlier kernels write are not `const
// __restrict__`: that would promise that the data does not change while the
// kernel runs (reads through the read-only path), and it runs before they end.
#pragma once
#include <cuda_runtime.h>

namespace clad3dgs {

__device__ __forceinline__ void wait_before() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
}

template <class... P, class... A>
cudaError_t launch_after(void (*kernel)(P...), unsigned grid, unsigned threads, size_t shared,
                         cudaStream_t stream, A&&... arguments) {
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(grid);
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = shared;
  config.stream = stream;
  config.attrs = &attribute;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kernel, P(arguments)...);
}

}  // namespace clad3dgs
