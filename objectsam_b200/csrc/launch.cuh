// Launches of the token operators' kernels.
#pragma once
#include <cuda_runtime.h>

#include <utility>

namespace osam {

// With the programmatic-serialization attribute a kernel may be scheduled while the one in front of it drains; it waits
// for that kernel's end (grid_dep_wait) before its first global access.  Two do not, and have their reasons: k_adamw reads
// its table before it, which is written once, when the plan is made, by a copy that no kernel starts ahead of; the dQ pass
// behind dK and dV (`late`) reads inputs and row terms at once, which were complete before any CTA in front let it start,
// writes what that pass does not touch, and waits at its end.
template <typename... P, typename... A>
cudaError_t launch_dependent(void (*k)(P...), unsigned grid, unsigned threads, size_t smem, cudaStream_t st, A&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k, std::forward<A>(args)...);
}

}  // namespace osam
