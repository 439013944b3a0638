// Launches that start while the kernel before them on the stream still runs (programmatic dependent launch).  A kernel that is launched so waits
// (pdl_wait) in every thread before it reads or writes anything that a kernel before may still use, and before it ends: then whoever waits for it
// waits for all that came before it as well.
#pragma once
#include "bw_common.cuh"

namespace bw {

__device__ __forceinline__ void pdl_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// `cluster`: CTAs of a cluster.
template <typename Kern, typename... Args>
int launch_early(const char *name, Kern kern, dim3 grid, int threads, int smem, cudaStream_t st, dim3 cluster, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cluster.x * cluster.y * cluster.z > 1) {
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = cluster.x;
        attr[1].val.clusterDim.y = cluster.y;
        attr[1].val.clusterDim.z = cluster.z;
        cfg.numAttrs = 2;
    }
    BW_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, args...));
    return check_launch(name);
}

}  // namespace bw
