// Sums over the threads that hold a row, for the kernels of the norms.
#pragma once

#include <hip/hip_runtime.h>

namespace osm {

// v plus its value in another lane of the 16: quads' pairs, halves, mirrors.
template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float lane_of(float v, int l) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l));
}
// The sum over 16 lanes, and over a wave, in every one of them: by DPP, then four
// scalars (a shuffle through LDS a step takes five times as long).
__device__ __forceinline__ float lanes_total(float v) {
  v = dpp_add<0xb1>(v);      // quad_perm 1 0 3 2
  v = dpp_add<0x4e>(v);      // quad_perm 2 3 0 1
  v = dpp_add<0x141>(v);     // row_half_mirror
  return dpp_add<0x140>(v);  // row_mirror
}
__device__ __forceinline__ float wave_total(float v) {
  v = lanes_total(v);
  return (lane_of(v, 0) + lane_of(v, 16)) + (lane_of(v, 32) + lane_of(v, 48));
}

// Sums over the TPR threads of a row, in every one of them.  `red`: one slot a
// wave and value; the caller's calls alternate its two halves.
template <int TPR, int K>
__device__ __forceinline__ void row_sum(float (&v)[K], float (*red)[K]) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = TPR == 16 ? lanes_total(v[k]) : wave_total(v[k]);
  if constexpr (TPR > 64) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) red[wave][k] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] = 0.0f;
#pragma unroll
      for (int w = 0; w < TPR / 64; ++w) v[k] += red[w][k];
    }
  }
}

}  // namespace osm
