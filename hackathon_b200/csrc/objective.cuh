// Shared by the preference and the policy objective: block sums in 64 bits. Both reduce masked
// [rows, cols] arrays to a handful of numbers in two launches: one CTA per (row, chunk of
// columns) writes a record of its sums, one CTA adds the records in a fixed order.
#pragma once

#include "qb_common.cuh"

namespace qb {

constexpr int kObjThreads = 256;
constexpr int kObjPerThread = 8;
constexpr int kObjChunk = kObjThreads * kObjPerThread;   // columns per CTA

// N sums over the block at once, in a fixed order; every thread gets them, or with FIRST only the
// first warp's. `scratch` holds 32 * N doubles.
template <bool FIRST = false, int N>
__device__ __forceinline__ void block_sums64(double (&v)[N], double* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int nwarps = (blockDim.x + 31) >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  __syncthreads();  // scratch may still be read by a previous call
  if (lane == 0)
#pragma unroll
    for (int k = 0; k < N; ++k) scratch[k * 32 + warp] = v[k];
  __syncthreads();
  if (FIRST && warp != 0) return;
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = lane < nwarps ? scratch[k * 32 + lane] : 0.0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
}

__device__ __forceinline__ double block_sum64(double v, double* scratch) {
  double a[1] = {v};
  block_sums64(a, scratch);
  return a[0];
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
