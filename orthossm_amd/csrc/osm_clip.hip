// The 2-norm over many tensors, and their scaling to a largest norm, on gfx950.
//
//   norm = sqrt(sum over all elements of all tensors of x^2)
//   x   <- x min(1, max_norm / (norm + eps))
//
// Two launches for a table of up to 150 tensors, whatever their sizes: the sums
// of squares over chunks of 8192 elements, then the scaling, every workgroup of
// which adds the (at most 1024 a table) partial sums itself, in order, so that
// no launch or atomic stands between.  Squares of fp32 and their sums are held
// in double: no overflow or underflow of a square, and the norm does not depend
// on the order of the additions beyond its last bit.  What bounds them: the
// bytes, read twice and written once; the scaling walks the chunks from the
// last to the first, so that what the caches still hold of the first pass is
// read from there.  Where the norm is within the limit nothing is written.
#include <algorithm>

#include "osm_norm.h"

namespace osm {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kThreads = 256;

// The tensor of a chunk.
__device__ __forceinline__ int tensor_of(const ClipTable& t, int chunk) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= chunk)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ double block_sum(double v, double* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

__global__ void __launch_bounds__(kThreads) clip_sums_kernel(const ClipTable t, double* part) {
  __shared__ double red[kThreads / 64];
  const int chunks = t.first[t.count];
  double sum = 0.0;
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int i = tensor_of(t, c);
    const int64_t e0 = (int64_t)(c - t.first[i]) * kClipChunk;
    const int n = (int)min((int64_t)kClipChunk, t.n[i] - e0);
    if (t.bf16[i]) {
      const __bf16* const x = static_cast<const __bf16*>(t.p[i]) + e0;
      int e = 8 * threadIdx.x;
      if (t.vec[i])
        for (; e + 8 <= n; e += 8 * kThreads) {
          const bf16x8 v = *reinterpret_cast<const bf16x8*>(x + e);
#pragma unroll
          for (int k = 0; k < 8; ++k) sum = __builtin_fma((double)(float)v[k], (double)(float)v[k], sum);
        }
      for (; e < n; e += 8 * kThreads)
        for (int k = e; k < min(e + 8, n); ++k) sum = __builtin_fma((double)(float)x[k], (double)(float)x[k], sum);
    } else {
      const float* const x = static_cast<const float*>(t.p[i]) + e0;
      int e = 4 * threadIdx.x;
      if (t.vec[i])
        for (; e + 4 <= n; e += 4 * kThreads) {
          const f32x4 v = *reinterpret_cast<const f32x4*>(x + e);
#pragma unroll
          for (int k = 0; k < 4; ++k) sum = __builtin_fma((double)v[k], (double)v[k], sum);
        }
      for (; e < n; e += 4 * kThreads)
        for (int k = e; k < min(e + 4, n); ++k) sum = __builtin_fma((double)x[k], (double)x[k], sum);
    }
  }
  sum = block_sum(sum, red);
  if (threadIdx.x == 0) part[t.part0 + blockIdx.x] = sum;
}

template <bool SCALE>
__global__ void __launch_bounds__(kThreads) clip_scale_kernel(const ClipTable t, const double* part, int parts,
                                                              double max_norm, double eps, float* norm) {
  __shared__ double red[kThreads / 64];
  double sum = 0.0;
  for (int i = threadIdx.x; i < parts; i += kThreads) sum += part[i];
  const double all = sqrt(block_sum(sum, red));
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)all;
  if (!SCALE) return;
  const float f = (float)(max_norm / (all + eps));
  if (f >= 1.0f) return;   // (a NaN norm goes on, and makes every element NaN)
  const int chunks = t.first[t.count];
  for (int c = chunks - 1 - blockIdx.x; c >= 0; c -= gridDim.x) {
    const int i = tensor_of(t, c);
    const int64_t e0 = (int64_t)(c - t.first[i]) * kClipChunk;
    const int n = (int)min((int64_t)kClipChunk, t.n[i] - e0);
    if (t.bf16[i]) {
      __bf16* const x = static_cast<__bf16*>(t.p[i]) + e0;
      int e = 8 * threadIdx.x;
      if (t.vec[i])
        for (; e + 8 <= n; e += 8 * kThreads) {
          bf16x8 v = *reinterpret_cast<const bf16x8*>(x + e);
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] = (__bf16)((float)v[k] * f);
          *reinterpret_cast<bf16x8*>(x + e) = v;
        }
      for (; e < n; e += 8 * kThreads)
        for (int k = e; k < min(e + 8, n); ++k) x[k] = (__bf16)((float)x[k] * f);
    } else {
      float* const x = static_cast<float*>(t.p[i]) + e0;
      int e = 4 * threadIdx.x;
      if (t.vec[i])
        for (; e + 4 <= n; e += 4 * kThreads) {
          f32x4 v = *reinterpret_cast<const f32x4*>(x + e);
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] *= f;
          *reinterpret_cast<f32x4*>(x + e) = v;
        }
      for (; e < n; e += 4 * kThreads)
        for (int k = e; k < min(e + 4, n); ++k) x[k] *= f;
    }
  }
}

}  // namespace

hipError_t launch_clip_sums(const ClipTable& t, double* part, hipStream_t stream) {
  hipLaunchKernelGGL(clip_sums_kernel, dim3(t.parts), dim3(kThreads), 0, stream, t, part);
  return hipGetLastError();
}

hipError_t launch_clip_scale(const ClipTable& t, const double* part, int parts, double max_norm, double eps, float* norm,
                             bool scale, hipStream_t stream) {
  if (scale)
    hipLaunchKernelGGL(clip_scale_kernel<true>, dim3(t.parts), dim3(kThreads), 0, stream, t, part, parts, max_norm, eps,
                       norm);
  else
    hipLaunchKernelGGL(clip_scale_kernel<false>, dim3(1), dim3(kThreads), 0, stream, t, part, parts, max_norm, eps, norm);
  return hipGetLastError();
}

}  // namespace osm
