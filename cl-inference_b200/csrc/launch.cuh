// launch.cuh -- kernel launches with the attributes the 8-bit operators use.
#pragma once

#include <cuda_runtime.h>

#include "clq_internal.h"

namespace clq {
namespace pipe {

// KERN<<<GRID, THREADS, SMEM, S>>>(ARGS...) in clusters of CLUSTER CTAs along x,
// a programmatic dependent launch unless CLQ_PDL=0.
template <typename... Args, typename... Given>
cudaError_t launch_cluster(void (*kern)(Args...), dim3 grid, int threads, size_t smem, int cluster, cudaStream_t s,
                           const Given&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    cfg.attrs = attr;
    if (gemv_pdl_enabled()) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = (unsigned)cluster;
        attr[cfg.numAttrs].val.clusterDim.y = 1;
        attr[cfg.numAttrs++].val.clusterDim.z = 1;
    }
    return cudaLaunchKernelEx(&cfg, kern, args...);
}
template <typename... Args, typename... Given>
cudaError_t launch_pdl(void (*kern)(Args...), dim3 grid, int threads, size_t smem, cudaStream_t s, const Given&... args) {
    return launch_cluster(kern, grid, threads, smem, 1, s, args...);
}

}  // namespace pipe
}  // namespace clq
