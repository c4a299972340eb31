// Shared by the preference and the policy objective: block sums in 64 bits. Both reduce masked
// [rows, cols] arrays to a handful of numbers in two launches: one CTA per (row, chunk of
// columns) writes a record of its sums, one CTA adds the records in a fixed order.
#pragma once

#include "qb_common.cuh"

namespace qb {

constexpr int kObjThreads = 256;
constexpr int kObjPerThread = 8;
constexpr int kObjChunk = kObjThreads * kObjPerThread;   // columns per CTA

__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum over the block in a fixed order; every thread gets it. `scratch` holds 32 doubles.
__device__ __forceinline__ double block_sum64(double v, double* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int nwarps = (blockDim.x + 31) >> 5;
  v = warp_sum64(v);
  __syncthreads();  // scratch may still be read by a previous call
  if (lane == 0) scratch[warp] = v;
  __syncthreads();
  return warp_sum64(lane < nwarps ? scratch[lane] : 0.0);
}

// Lanes that share a row's records in the adding CTA: a power of two, so that a row of few
// chunks takes few lanes (many rows at once) and a row of many is read by a whole warp.
inline int lanes_per_row(int chunks) {
  int lanes = 1;
  while (lanes < 32 && lanes < chunks) lanes *= 2;
  return lanes;
}

// Sum over the `lanes` consecutive lanes of a group; every lane of the group gets it. All lanes
// of the warp take part.
__device__ __forceinline__ double group_sum64(double v, int lanes) {
  for (int o = lanes / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Threads of the adding CTA for `rows` rows of `lanes` lanes each.
inline int adding_threads(int64_t rows, int lanes) {
  const int64_t want = rows > 1024 / lanes ? 1024 : (rows * lanes + 31) / 32 * 32;
  return static_cast<int>(want);
}

}  // namespace qb
