// Launches of the expert kernels.  A layer is a chain of short kernels on one stream: each is launched as a programmatic dependent of
// the one before, so that its blocks are placed, its barriers and tensor memory set up and its tensor maps
// fetched while the last blocks of that one still run.
// Inputs are not declared const __restrict__: the compiler may take such memory for constant over the whole kernel and move its
// loads above the wait.
// Every kernel here calls dependency_wait() in every thread before it touches global memory (it returns when the kernels before
// have finished and their results are visible), and dependents_go() once it holds all it needs of its SM - after
// tensor memory has been allocated: a dependent's block could otherwise take it first and both would wait for good.
#pragma once

#include "asp_internal.h"

namespace asp {

__device__ __forceinline__ void dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void dependents_go() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... P, typename... A>
alphasparseStatus_t launch_chained(alphasparseHandle_t h, void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, int cluster, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = h->stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = cluster;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  ASP_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
  ++impl(h)->launches;
  return ALPHA_SPARSE_STATUS_SUCCESS;
}

}  // namespace asp
