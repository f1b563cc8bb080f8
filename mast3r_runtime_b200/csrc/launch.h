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

}  // namespace m3r
