// Device code that layer normalisation and its gradient share.
#pragma once
#include "dense.h"

namespace hctr {

// The sum of v over the NT threads of a block, the same in all of them.  `smem` needs NT / 64 floats; the barriers inside keep
// one sum's words apart from the next one's.
template <int NT> __device__ __forceinline__ float block_sum(float v, float *smem) {
#pragma unroll
  for (int d = kWave / 2; d; d >>= 1) v += __shfl_xor(v, d, kWave);
  __syncthreads();
  if (lane_id() == 0) smem[threadIdx.x / kWave] = v;
  __syncthreads();
  v = 0.f;
#pragma unroll
  for (int i = 0; i < NT / kWave; i++) v += smem[i];
  return v;
}

// columns of weight or bias: `narrow`, they are of type A, else float; without any, `none`
template <int V, typename A>
__device__ __forceinline__ Floats<V> load_affine(const void *p, bool narrow, uint32_t c, uint32_t width, float none) {
  if (!p) {
    Floats<V> f;
#pragma unroll
    for (int j = 0; j < V; j++) f.v[j] = none;
    return f;
  }
  return narrow ? load_columns<V>((const A *)p, c, width) : load_columns<V>((const float *)p, c, width);
}

} // namespace hctr
