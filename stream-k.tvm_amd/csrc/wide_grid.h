// Blocks of one-dimensional work where there may be so many that their threads no longer count in 32 bits, which no launch takes in one
// dimension (2^24 rows of 256 threads): the numbers go on in the grid's second dimension.  The last row of the grid may have blocks too many.
#pragma once
#include <hip/hip_runtime.h>

namespace sk {

constexpr int WIDE_GRID_BITS = 21;   // (blocks of up to 1024 threads)
static inline dim3 wide_grid(int64_t blocks) {
  const int64_t most = (int64_t)1 << WIDE_GRID_BITS;
  return blocks <= most ? dim3((unsigned)blocks) : dim3((unsigned)most, (unsigned)((blocks + most - 1) >> WIDE_GRID_BITS));
}
__device__ __forceinline__ int64_t wide_block() { return ((int64_t)blockIdx.y << WIDE_GRID_BITS) + blockIdx.x; }

}  // namespace sk
