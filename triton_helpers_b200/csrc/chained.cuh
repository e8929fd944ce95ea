// Launches that overlap their start with the end of the kernel before (programmatic dependent launch).  Each kernel of the wide layers lets
// the next one start (start_next) and touches no global memory before the kernels ahead of it have finished (after_previous): what overlaps is
// the launch and the set-up of barriers, tensor memory and descriptors.  A neighbour that knows nothing of this runs strictly before or after.
//
// One exception: a product that is told so (GemmArgs::early) fetches weights ahead of its wait.  It may only because the kernel ahead of it, which
// makes 8-bit rows (row_fwd_kernel, row_fwd_stream_kernel), lets it start after its own wait and not before, so that whatever wrote the weights
// has finished by then.  All other kernels let the next one start at once.
#pragma once

#include "common.cuh"

namespace th {
namespace {

__device__ __forceinline__ void start_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... Params, typename... Args>
int launch_chained(const char *what, void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, unsigned cluster, Args &&...args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attrs[2]{};
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.x = cluster;
    attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
    cfg.attrs = attrs;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
    note_launch();
    return cuda_status(err, what);
}

}  // namespace
}  // namespace th
