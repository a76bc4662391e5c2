// Kernels that follow one another on a stream, as an expert layer's do: the next one is launched while the last
// CTAs of the previous one still run, sets up (barriers, tensor memory, instruction fetch) and waits
// before it touches memory. Worth about two microseconds per kernel boundary.
//
// Rules that make it safe: a kernel calls chain_wait() in every CTA before its first access to global
// memory (its predecessor has then finished, and with it everything before that), and chain_next() only
// once the CTA holds all it has to allocate (tensor memory above all): a CTA of the next kernel may
// take what is left, and must never be what this kernel waits for.
#pragma once
#include <cuda_runtime.h>

namespace b200dq {

__device__ __forceinline__ void chain_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void chain_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// kernel<<<grid, threads, smem, stream>>>(args...), allowed to start under its predecessor's end; clusters of
// `cluster` CTAs.
template <typename... Params, typename... Args>
cudaError_t chain_launch(void (*kernel)(Params...), unsigned grid, unsigned threads, size_t smem, cudaStream_t stream,
                         unsigned cluster, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
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
  cfg.numAttrs = cluster > 0 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}

}  // namespace b200dq
