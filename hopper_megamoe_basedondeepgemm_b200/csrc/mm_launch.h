// A launch that may begin before the kernel ahead of it in its stream has ended: its launch and the part of it before `grid_dependency_wait` overlap with that kernel's
// end. What that kernel wrote is there after the wait. A kernel launched so lets the next one in (`grid_launch_dependents`) only behind its own wait: then whatever
// runs early has at most one kernel of its stream ahead of it that has not ended, and waits for that one.
#pragma once
#include <cuda_runtime.h>

namespace mm {

template <typename P>
cudaError_t launch_behind(void (*kernel)(P), unsigned grid, unsigned threads, cudaStream_t stream, const P& params) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid); cfg.blockDim = dim3(threads); cfg.stream = stream;
    cfg.attrs = attr; cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, params);
}

// A launch that begins when the kernel ahead of it has ended. Like those above it says how it went by itself: `cudaGetLastError` would report what an earlier call left.
template <typename... P, typename... A>
cudaError_t launch_plain(void (*kernel)(P...), unsigned grid, unsigned threads, cudaStream_t stream, A&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid); cfg.blockDim = dim3(threads); cfg.stream = stream;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

// Clusters of `size` CTAs (at most eight), as early.
template <typename P>
cudaError_t launch_clusters(void (*kernel)(P), unsigned grid, unsigned size, unsigned threads, cudaStream_t stream, const P& params) {
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = size; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid); cfg.blockDim = dim3(threads); cfg.stream = stream;
    cfg.attrs = attr; cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, params);
}

}  // namespace mm
