// Launches that overlap their start with the end of the kernel before (programmatic dependent launch).  Each kernel of the wide layers waits for
// the kernels ahead of it before it touches global memory, and lets the next one start after that wait (after_previous does both): what overlaps is
// the launch and the set-up of barriers, tensor memory and descriptors.  A neighbour that knows nothing of this runs strictly before or after.
//
// The order matters.  CTAs that have started early hold registers, shared memory and tensor memory while they wait, so they must only wait for a kernel
// that needs no more of these: when its successor starts, all CTAs of a kernel have started, have their tensor memory and are past their own wait.
//
// One access comes ahead of the wait: a product that is told so (GemmArgs::early) fetches its first weights.  It may because whatever was launched
// before the kernel ahead had finished when that one passed its wait.
#pragma once

#include "common.cuh"

namespace th {
namespace {

// By all threads of the CTA
__device__ __forceinline__ void after_previous() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __syncthreads();  // all of them are past it
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

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
