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
// read from there: 56 tensors of 218 MB, from memory, take 48 us for the norm and 114
// with the scaling (4.6 and 5.8 TB/s).  Where the norm is within the limit nothing is
// written.
#include <algorithm>

#include "osm_norm.h"
#include "osm_wide_store.h"

namespace osm {
namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

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

// A chunk's place, and its elements where it is whole and aligned: 4 (bf16) or 8
// (fp32) loads of 16 bytes a thread, all of them on their way at once.
struct Chunk {
  char* x;
  int n;
  bool bf16, whole;
  u32x4 v[8];

  __device__ __forceinline__ void load(const ClipTable& t, int c) {
    const int i = tensor_of(t, c);
    const int64_t e0 = (int64_t)(c - t.first[i]) * kClipChunk;
    bf16 = t.bf16[i];
    x = static_cast<char*>(t.p[i]) + e0 * (bf16 ? 2 : 4);
    n = (int)min((int64_t)kClipChunk, t.n[i] - e0);
    whole = n == kClipChunk && t.vec[i];
    if (!whole) return;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < 4 || !bf16) v[k] = *reinterpret_cast<const u32x4*>(x + at(k));
  }
  __device__ __forceinline__ static unsigned at(int k) { return 16u * (k * kThreads + threadIdx.x); }
};

__device__ __forceinline__ void add_square(double& sum, float x) { sum = __builtin_fma((double)x, (double)x, sum); }
__device__ __forceinline__ float low(unsigned v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float high(unsigned v) { return __uint_as_float(v & 0xffff0000u); }

__device__ __forceinline__ void add_squares(double (&sum)[2], const Chunk& c) {
  if (!c.whole) {
    for (int e = threadIdx.x; e < c.n; e += kThreads)
      add_square(sum[0], c.bf16 ? (float)reinterpret_cast<const __bf16*>(c.x)[e] : reinterpret_cast<const float*>(c.x)[e]);
  } else if (c.bf16) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        add_square(sum[0], low(c.v[k][i]));
        add_square(sum[1], high(c.v[k][i]));
      }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) add_square(sum[i & 1], __uint_as_float(c.v[k][i]));
  }
}

// A workgroup loads its next chunk before it adds up the one it has.
__global__ void __launch_bounds__(kThreads) clip_sums_kernel(const ClipTable t, double* part) {
  __shared__ double red[kThreads / 64];
  const int chunks = t.first[t.count], turn = gridDim.x;
  double sum[2] = {0.0, 0.0};
  Chunk a, b;
  int c = blockIdx.x;
  if (c < chunks) a.load(t, c);
  while (c < chunks) {
    if (c + turn < chunks) b.load(t, c + turn);
    add_squares(sum, a);
    if (c + turn >= chunks) break;
    if (c + 2 * turn < chunks) a.load(t, c + 2 * turn);
    add_squares(sum, b);
    c += 2 * turn;
  }
  const double all = block_sum(sum[0] + sum[1], red);
  if (threadIdx.x == 0) part[t.part0 + blockIdx.x] = all;
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
  for (int i = chunks - 1 - blockIdx.x; i >= 0; i -= gridDim.x) {
    Chunk c;
    c.load(t, i);
    if (!c.whole) {
      for (int e = threadIdx.x; e < c.n; e += kThreads) {
        if (c.bf16) {
          __bf16* const x = reinterpret_cast<__bf16*>(c.x) + e;
          *x = (__bf16)((float)*x * f);
        } else {
          reinterpret_cast<float*>(c.x)[e] *= f;
        }
      }
      continue;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (k >= 4 && c.bf16) break;
      u32x4 v = c.v[k];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[i] = c.bf16 ? __builtin_bit_cast(unsigned, bf16x2{(__bf16)(low(v[i]) * f), (__bf16)(high(v[i]) * f)})
                      : __float_as_uint(__uint_as_float(v[i]) * f);
      *reinterpret_cast<u32x4*>(c.x + Chunk::at(k)) = v;
      wide_store_wait();
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
