// The output columns that a warp of the few-row product works through.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define M3R_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define M3R_HOST_DEVICE inline
#endif

namespace m3r {

// Groups of columns from `at` on, `step` apart, below n.  Unsigned: n is below 2^31, but the step past the
// last group may reach beyond it (a grid of 148 x 2 blocks steps 9,472 columns), which a signed index
// would turn into a column in front of the matrix.
struct ColumnWalk {
    uint32_t at, step, n;
    M3R_HOST_DEVICE bool live() const { return at < n; }
    M3R_HOST_DEVICE void next() { at += step; }
    // column i of the group; the last one for those past the end
    M3R_HOST_DEVICE uint32_t column(uint32_t i) const { return at + i < n ? at + i : n - 1; }
};

}  // namespace m3r
