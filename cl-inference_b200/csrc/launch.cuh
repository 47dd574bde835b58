// launch.cuh -- kernel launches with the attributes the 8-bit operators use.
#pragma once

#include <atomic>
#include <cstdint>

#include <cuda_runtime.h>

#include "clq_internal.h"

namespace clq {
namespace pipe {

constexpr size_t kSmemPerSm = 227 * 1024;  // of one CTA at most

// Opts KERN into SMEM bytes of shared memory, once per device (a decoded
// token's call takes a few microseconds, and the driver call is one of them).
template <typename Kern>
cudaError_t allow_smem(Kern kern, size_t smem, std::atomic<uint64_t>& done) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
    return e;
}

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
