// A workgroup's inclusive prefix sum, for the kernels that find their work in a list of lengths on the device.
#pragma once

#include <stddef.h>

#include "dsa_common.h"

namespace dsa {

// v's inclusive prefix sum over the THREADS threads of the workgroup (all of them call it), and its total; tot: THREADS /
// WAVE ints of LDS.
template <int THREADS>
__device__ __forceinline__ int group_incl_scan(int v, int* tot, int& total) {
  const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
  const int x = wave_incl_scan(v);
  __syncthreads();  // (tot's earlier readers)
  if (lane == WAVE - 1) tot[wave] = x;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / WAVE; ++w) {
    const int s = tot[w];
    before += w < wave ? s : 0;
    total += s;
  }
  return before + x;
}

}  // namespace dsa
