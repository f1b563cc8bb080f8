// Launch helpers of the operators.
#pragma once

#include <cuda_runtime.h>

#include <mutex>

#include "tmap.h"

namespace m3r {

// Raises a kernel's shared memory limit once on each device; `done` holds the devices (one word for
// each kernel).  Always to the same value, so that concurrent calls cannot lower it.
template <class Kernel>
void allow_smem(Kernel kern, int bytes, unsigned& done) {
    int dev = 0;
    M3R_CUDA(cudaGetDevice(&dev));
    static std::mutex mu;
    std::lock_guard<std::mutex> lock(mu);
    if (dev < 32 && (done >> dev & 1)) return;
    M3R_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    if (dev < 32) done |= 1u << dev;
}

// A launch that may start before the kernel ahead of it on the stream has finished (the kernel keeps the
// rules of common.cuh: grid_dependency_wait before it touches memory, plain loads), which hides its start
// behind that one's end (24 x 4,096 x 4,096 with its quantisation, one call after the other: 10.2 us
// against 8.4); cluster size 0: none.  With `dependent` false, an ordinary launch.  Launched with
// cudaLaunchKernelEx either way, whose status is this launch's own: cudaGetLastError would also give an error
// that an earlier call of the thread left.
struct LaunchConfig {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    LaunchConfig(unsigned grid, int block, int smem, cudaStream_t s, int cluster = 0, bool dependent = true) {
        cfg.gridDim = dim3(grid);
        cfg.blockDim = dim3(block);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = s;
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = cluster;
        attr[1].val.clusterDim.y = 1;
        attr[1].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = cluster > 0 ? 2 : dependent ? 1 : 0;
    }
    LaunchConfig(const LaunchConfig&) = delete;
};

}  // namespace m3r
