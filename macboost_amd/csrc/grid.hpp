// grid.hpp — grids of more workgroups than HIP takes along x, where a launch may have
// fewer than 2^32 threads: runs of 2^23 workgroups lie along z.
#pragma once
#include <hip/hip_runtime.h>

namespace mbk {

constexpr int64_t GRID_X = (int64_t)1 << 23;     // of up to 256 threads
inline dim3 grid_of(int64_t groups, uint32_t y = 1) {
    if (groups <= GRID_X) return dim3((uint32_t)groups, y);
    return dim3((uint32_t)GRID_X, y, (uint32_t)((groups + GRID_X - 1) / GRID_X));
}
// The last run may have workgroups behind the end.
__device__ __forceinline__ uint32_t group_id() { return blockIdx.z * gridDim.x + blockIdx.x; }
__device__ __forceinline__ uint32_t group_count() { return gridDim.z * gridDim.x; }

}  // namespace mbk
