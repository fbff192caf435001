// Launches that may be queued on the SMs while the kernel in front of them in the stream drains
// (programmatic dependent launch): a kernel launched with launch_dependent calls dependent_start()
// before it touches global memory, which waits until the kernels before it are complete and their
// writes visible, and lets the one behind it be queued in turn.  The order of the stream is kept; what
// is hidden is the launch itself, 1-2 us a call.  Such a kernel reads its inputs with plain loads or
// load16: the read-only path (__ldg, const __restrict__) is for data that nobody writes during the
// kernel's life, which here begins before the wait.
#pragma once

#include "hl_common.cuh"

namespace hl {

__device__ __forceinline__ void dependent_start() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// 16 bytes from L2, past L1; not moved in front of dependent_start.  (Plain 16-byte loads in its place:
// 20.1 against 17.6 us for a store of 8195 tokens.)
__device__ __forceinline__ uint4 load16(const void* p) {
  uint4 v;
  asm volatile("ld.global.cg.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// cluster: thread blocks per cluster (1: none).
template <typename... Params, typename... Args>
cudaError_t launch_dependent(void (*kernel)(Params...), dim3 grid, int threads, size_t shared, int cluster,
                             cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = shared;
  cfg.stream = stream;
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = cluster;
  attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
  cfg.attrs = attrs;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, Params(args)...);
}

}  // namespace hl
