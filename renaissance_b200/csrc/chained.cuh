// Launches that overlap the end of the kernel before them on the stream (programmatic dependent launch).
#pragma once

#include <cuda_runtime.h>

namespace trb {
namespace ptx {

// For kernels launched by launch_chained(): everything before wait_prior_grid() may run while the kernel before on the
// stream still does, so nothing is read or written before it; let_next_grid_start() by all blocks lets the next one in.
__device__ __forceinline__ void wait_prior_grid() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_grid_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

}  // namespace ptx

// The kernel begins with wait_prior_grid().  `cluster` blocks in x form a cluster.
template <class... Par, class... Arg>
cudaError_t launch_chained(void (*kernel)(Par...), unsigned grid, unsigned block, unsigned cluster, size_t smem, cudaStream_t s, Arg... arg) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, Par(arg)...);
}

}  // namespace trb
