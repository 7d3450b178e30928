// Layer norm on gfx950, forward and backward.
//
//   mean = sum x / D,  rstd = 1 / sqrt(sum (x - mean)^2 / D + eps)
//   y = xh w + b,  xh = (x - mean) rstd
//   dx = rstd (w dy - mean(w dy) - xh mean(w dy xh)),  dw = sum_rows dy xh,  db = sum_rows dy
//
// A row is held in the registers of one wave, of a quarter of one where it is
// short, or of four or sixteen where it is longer, so x is read once in each direction and the variance is a second sum
// over registers, free of cancellation.  What bounds both: the bytes of x, y
// (x, dy, dx); 262144 bf16 rows of 1024 take 206 us forward and 273 backward (5.2
// and 5.9 TB/s).  The backward's workgroups walk rows a grid apart and keep their
// columns' sums of dy xh and dy in registers; each writes one line of partial
// sums, which a second launch adds in order, so the result does not depend on
// timing.  Rows too long for registers are read again for each sum.
#include <algorithm>
#include <type_traits>

#include "osm_norm.h"
#include "osm_wide_store.h"

// Fused multiply-adds are written where they are meant: w dy - mean as one
// would leave the rounding of w dy in a dx that is 0 (rows of one element).
#pragma clang fp contract(off)

namespace osm {
namespace {

template <typename T>
constexpr int kUnit = 16 / (int)sizeof(T);   // elements of a 16-byte access

// 16 bytes of a row as loaded, and their values.  Rows that do not start at multiples
// of 16 bytes are read and written by the same pieces at an element's alignment, but
// for their ends (2^26 bf16 elements in rows of 1001, element by element against so:
// forward 165 and 70 us, backward 348 and 116).
template <typename T>
struct Unit {
  typedef T Vec __attribute__((ext_vector_type(kUnit<T>)));
  typedef T Loose __attribute__((ext_vector_type(kUnit<T>), aligned(sizeof(T))));
  Vec raw;
  __device__ __forceinline__ void get(float (&v)[kUnit<T>]) const {
#pragma unroll
    for (int i = 0; i < kUnit<T>; ++i) v[i] = (float)raw[i];
  }
};

template <typename T>
__device__ __forceinline__ void store_unit(T* p, const float (&v)[kUnit<T>]) {
  typename Unit<T>::Vec q;
#pragma unroll
  for (int i = 0; i < kUnit<T>; ++i) q[i] = (T)v[i];
  __builtin_nontemporal_store(q, reinterpret_cast<typename Unit<T>::Vec*>(p));
  wide_store_wait();
}

// A row's units u, u + TPR, .. of a thread; past the row's end: zeros, and no
// stores.  vec: rows start at multiples of 16 bytes and D is whole units.
template <typename T, int TPR, int NV>
struct Row {
  static constexpr int U = kUnit<T>;
  // As loaded, so that the next row can be on its way while this one is worked on.
  struct Raw {
    Unit<T> n[NV];
    __device__ __forceinline__ void load(const T* p, int D, int u, bool vec) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (u + k * TPR) * U;
        typename Unit<T>::Vec v = {};
        if (vec) {
          if (c < D) v = __builtin_nontemporal_load(reinterpret_cast<const typename Unit<T>::Vec*>(p + c));
        } else if (c + U <= D) {   // (whole, at an element's alignment)
          v = *reinterpret_cast<const typename Unit<T>::Loose*>(p + c);
        } else {
#pragma unroll
          for (int i = 0; i < U; ++i)
            if (c + i < D) v[i] = p[c + i];
        }
        n[k].raw = v;
      }
    }
    __device__ __forceinline__ void get(float (&v)[NV][U]) const {
#pragma unroll
      for (int k = 0; k < NV; ++k) n[k].get(v[k]);
    }
  };
  static __device__ __forceinline__ void store(T* p, const float (&v)[NV][U], int D, int u, bool vec) {
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int c = (u + n * TPR) * U;
      if (vec) {
        if (c < D) store_unit<T>(p + c, v[n]);
      } else if (c + U <= D) {
        typename Unit<T>::Vec q;
#pragma unroll
        for (int i = 0; i < U; ++i) q[i] = (T)v[n][i];
        *reinterpret_cast<typename Unit<T>::Loose*>(p + c) = q;
        wide_store_wait();
      } else {
#pragma unroll
        for (int i = 0; i < U; ++i)
          if (c + i < D) p[c + i] = (T)v[n][i];
      }
    }
  }
  // fp32 parameters of the same columns; `fill` where there are none
  static __device__ __forceinline__ void param(float (&v)[NV][U], const float* w, float fill, int D, int u) {
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int c = (u + n * TPR) * U + i;
        v[n][i] = c < D ? (w ? w[c] : fill) : 0.0f;
      }
  }
};

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

// TPR threads a row, max(TPR, 256) a workgroup.
template <typename T, int TPR, int NV>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256) layer_norm_fwd_kernel(const NormParams p) {
  using R = Row<T, TPR, NV>;
  constexpr int kThreads = TPR > 256 ? TPR : 256, kRows = kThreads / TPR, U = R::U;
  __shared__ float red[2][kThreads / 64][1];
  const int u = threadIdx.x % TPR;
  float w[NV][U], b[NV][U], x[NV][U];
  R::param(w, p.weight, 1.0f, p.D, u);
  R::param(b, p.bias, 0.0f, p.D, u);
  // (every thread of a workgroup runs the same trips: kRows is 1 where row_sum has barriers)
  const int64_t step = (int64_t)gridDim.x * kRows;
  int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / TPR;
  typename R::Raw next;
  if (row < p.rows) next.load(static_cast<const T*>(p.x) + row * p.x_stride, p.D, u, p.vec);
  for (; row < p.rows; row += step) {
    next.get(x);
    if (row + step < p.rows) next.load(static_cast<const T*>(p.x) + (row + step) * p.x_stride, p.D, u, p.vec);
    float s[1] = {0.0f};
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
      for (int i = 0; i < U; ++i) s[0] += x[n][i];
    row_sum<TPR>(s, red[0]);
    const float mean = s[0] / (float)p.D;
    s[0] = 0.0f;
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
      for (int i = 0; i < U; ++i) {
        x[n][i] = (u + n * TPR) * U + i < p.D ? x[n][i] - mean : 0.0f;
        s[0] = __builtin_fmaf(x[n][i], x[n][i], s[0]);
      }
    row_sum<TPR>(s, red[1]);
    const float rstd = 1.0f / sqrtf(s[0] / (float)p.D + p.eps);
    if (p.mean && u == 0) {
      p.mean[row] = mean;
      p.rstd[row] = rstd;
    }
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
      for (int i = 0; i < U; ++i) x[n][i] = __builtin_fmaf(x[n][i] * rstd, w[n][i], b[n][i]);
    R::store(static_cast<T*>(p.y) + row * p.y_stride, x, p.D, u, p.vec);
  }
}

template <typename T, int TPR, int NV>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256) layer_norm_bwd_kernel(const NormParams p) {
  using R = Row<T, TPR, NV>;
  constexpr int kThreads = TPR > 256 ? TPR : 256, kRows = kThreads / TPR, U = R::U;
  __shared__ float red[2][kThreads / 64][2];
  const int u = threadIdx.x % TPR;
  float w[NV][U], dw[NV][U], db[NV][U], x[NV][U], g[NV][U];
  R::param(w, p.weight, 1.0f, p.D, u);
#pragma unroll
  for (int n = 0; n < NV; ++n)
#pragma unroll
    for (int i = 0; i < U; ++i) dw[n][i] = db[n][i] = 0.0f;
  int par = 0;
  const int64_t step = (int64_t)gridDim.x * kRows;
  int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / TPR;
  typename R::Raw next_x, next_g;
  float next_mean = 0.0f, next_rstd = 0.0f;
  auto fetch = [&](int64_t at) {
    next_x.load(static_cast<const T*>(p.x) + at * p.x_stride, p.D, u, p.vec);
    next_g.load(static_cast<const T*>(p.gy) + at * p.gy_stride, p.D, u, p.vec);
    next_mean = p.mean[at];
    next_rstd = p.rstd[at];
  };
  if (row < p.rows) fetch(row);
  for (; row < p.rows; row += step) {
    next_x.get(x);
    next_g.get(g);
    const float mean = next_mean, rstd = next_rstd;
    if (row + step < p.rows) fetch(row + step);
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const float xh = (x[n][i] - mean) * rstd;
        dw[n][i] = __builtin_fmaf(g[n][i], xh, dw[n][i]);
        db[n][i] += g[n][i];
        g[n][i] *= w[n][i];          // zeros past the row's end: w and g are
        x[n][i] = xh;
        s[0] += g[n][i];
        s[1] = __builtin_fmaf(g[n][i], xh, s[1]);
      }
    row_sum<TPR>(s, red[par]);
    par ^= 1;
    const float a = s[0] / (float)p.D, c = s[1] / (float)p.D;
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
      for (int i = 0; i < U; ++i) x[n][i] = rstd * (g[n][i] - a - x[n][i] * c);
    if (p.gx) R::store(static_cast<T*>(p.gx) + row * p.gx_stride, x, p.D, u, p.vec);
  }
  // This workgroup's line of sums: its row groups in order.
  float* const line = p.part + (int64_t)blockIdx.x * 2 * p.D;
  if constexpr (kRows > 1) {
    __shared__ float sums[kRows - 1][2][TPR * U];
    const int group = threadIdx.x / TPR;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      __syncthreads();
      if (group > 0)
#pragma unroll
        for (int i = 0; i < U; ++i) {
          sums[group - 1][0][i * TPR + u] = dw[n][i];
          sums[group - 1][1][i * TPR + u] = db[n][i];
        }
      __syncthreads();
      if (group == 0)
#pragma unroll 3
        for (int q = 0; q < kRows - 1; ++q)
#pragma unroll
          for (int i = 0; i < U; ++i) {
            dw[n][i] += sums[q][0][i * TPR + u];
            db[n][i] += sums[q][1][i * TPR + u];
          }
    }
    if (group > 0) return;
  }
#pragma unroll
  for (int n = 0; n < NV; ++n)
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int c = (u + n * TPR) * U + i;
      if (c < p.D) {
        line[c] = dw[n][i];
        line[p.D + c] = db[n][i];
      }
    }
}

constexpr int kLongThreads = 1024;

// Rows too long for registers: a workgroup a row, read again for every sum.
template <typename T>
__global__ void __launch_bounds__(kLongThreads) layer_norm_fwd_long_kernel(const NormParams p) {
  __shared__ float red[2][kLongThreads / 64][1];
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* const x = static_cast<const T*>(p.x) + row * p.x_stride;
    T* const y = static_cast<T*>(p.y) + row * p.y_stride;
    float s[1] = {0.0f};
    for (int64_t c = threadIdx.x; c < p.D; c += kLongThreads) s[0] += (float)x[c];
    row_sum<kLongThreads>(s, red[0]);
    const float mean = s[0] / (float)p.D;
    s[0] = 0.0f;
    for (int64_t c = threadIdx.x; c < p.D; c += kLongThreads) {
      const float d = (float)x[c] - mean;
      s[0] = __builtin_fmaf(d, d, s[0]);
    }
    row_sum<kLongThreads>(s, red[1]);
    const float rstd = 1.0f / sqrtf(s[0] / (float)p.D + p.eps);
    if (p.mean && threadIdx.x == 0) {
      p.mean[row] = mean;
      p.rstd[row] = rstd;
    }
    for (int64_t c = threadIdx.x; c < p.D; c += kLongThreads)
      y[c] = (T)__builtin_fmaf(((float)x[c] - mean) * rstd, p.weight ? p.weight[c] : 1.0f, p.bias ? p.bias[c] : 0.0f);
  }
}

// dx of long rows; their dw and db by columns (the next kernel).
template <typename T>
__global__ void __launch_bounds__(kLongThreads) layer_norm_bwd_long_kernel(const NormParams p) {
  __shared__ float red[2][kLongThreads / 64][2];
  int par = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* const x = static_cast<const T*>(p.x) + row * p.x_stride;
    const T* const gy = static_cast<const T*>(p.gy) + row * p.gy_stride;
    const float mean = p.mean[row], rstd = p.rstd[row];
    float s[2] = {0.0f, 0.0f};
    for (int64_t c = threadIdx.x; c < p.D; c += kLongThreads) {
      const float g = (float)gy[c] * (p.weight ? p.weight[c] : 1.0f);
      s[0] += g;
      s[1] = __builtin_fmaf(g, ((float)x[c] - mean) * rstd, s[1]);
    }
    row_sum<kLongThreads>(s, red[par]);
    par ^= 1;
    const float a = s[0] / (float)p.D, m = s[1] / (float)p.D;
    if (p.gx) {
      T* const gx = static_cast<T*>(p.gx) + row * p.gx_stride;
      for (int64_t c = threadIdx.x; c < p.D; c += kLongThreads) {
        const float g = (float)gy[c] * (p.weight ? p.weight[c] : 1.0f);
        gx[c] = (T)(rstd * (g - a - ((float)x[c] - mean) * rstd * m));
      }
    }
  }
}

// A line of sums of long rows: workgroup (columns, line) takes rows line,
// line + lines, ...
template <typename T>
__global__ void __launch_bounds__(256) layer_norm_columns_kernel(const NormParams p) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= p.D) return;
  float dw = 0.0f, db = 0.0f;
  for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
    const float g = (float)static_cast<const T*>(p.gy)[row * p.gy_stride + c];
    const float x = (float)static_cast<const T*>(p.x)[row * p.x_stride + c];
    dw = __builtin_fmaf(g, (x - p.mean[row]) * p.rstd[row], dw);
    db += g;
  }
  float* const line = p.part + (int64_t)blockIdx.y * 2 * p.D;
  line[c] = dw;
  line[p.D + c] = db;
}

constexpr int kFoldCols = 32, kFoldGroups = 32;

// dw and db from the lines, 32 columns a workgroup: group g adds lines g, g + 32,
// ..; then the groups in order.
__global__ void __launch_bounds__(kFoldCols * kFoldGroups) layer_norm_fold_kernel(const float* part, float* dw, float* db,
                                                                                  int64_t D, int lines) {
  __shared__ float red[kFoldGroups][kFoldCols];
  const int cl = threadIdx.x % kFoldCols, g = threadIdx.x / kFoldCols;
  const int64_t c = (int64_t)blockIdx.x * kFoldCols + cl;
  float s = 0.0f;
  if (c < 2 * D) {
#pragma unroll 8
    for (int i = g; i < lines; i += kFoldGroups) s += part[(int64_t)i * 2 * D + c];
  }
  red[g][cl] = s;
  __syncthreads();
  if (g == 0 && c < 2 * D) {
#pragma unroll
    for (int q = 1; q < kFoldGroups; ++q) s += red[q][cl];
    float* const dst = c < D ? dw : db;
    if (dst) dst[c < D ? c : c - D] = s;
  }
}

// Calls go(TPR, NV) for the fewest threads that hold a row, 16 elements each (LAST
// in the case of 1024 threads: the backward holds five rows' worth, and spills
// with 16), or long_rows() past 1024 LAST elements.  Measured with 64 and 256
// threads a row, forward and backward: bf16, 262144 rows of 1024 206 and 288 us, 298
// and 362; fp32, 15003 rows of 400 13 and 17 us, 18 and 24.  With 16 and 64, bf16,
// 2^26 elements in rows of 16 246 and 1038 us, 306 and 1206, of 64 65 and 257, 84 and
// 311; fp32, of 64 101 and 212, 143 and 256.
template <typename T, int LAST, typename Go, typename Long>
void by_length(int64_t D, Go go, Long long_rows) {
  const int64_t units = (D + kUnit<T> - 1) / kUnit<T>;
  auto pick = [&](auto tpr) {
    constexpr int TPR = decltype(tpr)::value, most = TPR == 16 ? 1 : (TPR == 1024 ? LAST : 16) / kUnit<T>;
    if (units > most * TPR) return false;
    if (units <= TPR)
      go(tpr, std::integral_constant<int, 1>{});
    else if (most == 2 || units <= 2 * TPR)
      go(tpr, std::integral_constant<int, most == 1 ? 1 : 2>{});
    else
      go(tpr, std::integral_constant<int, most>{});
    return true;
  };
  if (!pick(std::integral_constant<int, 16>{}) && !pick(std::integral_constant<int, 64>{}) &&
      !pick(std::integral_constant<int, 256>{}) && !pick(std::integral_constant<int, 1024>{}))
    long_rows();
}

constexpr int kMaxGroups = 2048;

template <typename T>
hipError_t forward(const NormParams& p, hipStream_t stream) {
  by_length<T, 16>(
      p.D,
      [&](auto tpr, auto nv) {
        constexpr int TPR = decltype(tpr)::value, NV = decltype(nv)::value, kThreads = TPR > 256 ? TPR : 256;
        const int64_t groups = (p.rows + kThreads / TPR - 1) / (kThreads / TPR);
        hipLaunchKernelGGL((layer_norm_fwd_kernel<T, TPR, NV>), dim3((unsigned)std::min<int64_t>(groups, kMaxGroups)),
                           dim3(kThreads), 0, stream, p);
      },
      [&] {
        hipLaunchKernelGGL((layer_norm_fwd_long_kernel<T>), dim3((unsigned)std::min<int64_t>(p.rows, kMaxGroups)),
                           dim3(kLongThreads), 0, stream, p);
      });
  return hipGetLastError();
}

template <typename T>
hipError_t backward(const NormParams& p, float* dw, float* db, hipStream_t stream) {
  const int lines = norm_lines(p.rows, p.D);
  hipError_t e = hipSuccess;
  by_length<T, 8>(
      p.D,
      [&](auto tpr, auto nv) {
        constexpr int TPR = decltype(tpr)::value, NV = decltype(nv)::value, kThreads = TPR > 256 ? TPR : 256;
        hipLaunchKernelGGL((layer_norm_bwd_kernel<T, TPR, NV>), dim3(lines), dim3(kThreads), 0, stream, p);
      },
      [&] {
        hipLaunchKernelGGL((layer_norm_bwd_long_kernel<T>), dim3((unsigned)std::min<int64_t>(p.rows, kMaxGroups)),
                           dim3(kLongThreads), 0, stream, p);
        e = hipGetLastError();
        if (e == hipSuccess)
          hipLaunchKernelGGL((layer_norm_columns_kernel<T>), dim3((unsigned)((p.D + 255) / 256), lines), dim3(256), 0,
                             stream, p);
      });
  if (e == hipSuccess) e = hipGetLastError();
  if (e != hipSuccess || (!dw && !db)) return e;
  hipLaunchKernelGGL(layer_norm_fold_kernel, dim3((unsigned)((2 * p.D + kFoldCols - 1) / kFoldCols)),
                     dim3(kFoldCols * kFoldGroups), 0, stream, p.part, dw, db, p.D, lines);
  return hipGetLastError();
}

}  // namespace

// Workgroups of the backward, and lines of partial sums: enough to fill the chip,
// few enough that the lines are a small part of the rows' bytes and that a
// workgroup's rows follow each other closely in memory.  Measured in us with 256,
// 512 and 1024 lines: bf16, 262144 rows of D=256 182, 114, 92, of 1024 282, 274, 298;
// 65536 of 4096 294, 283, 305; 4096 of 16384 243, 260, 294; 4096 of 1024 12.8, 14.9,
// 22.0; fp32, 2048 rows of 1024 10.3, 11.8, 11.9; 1024 of 65536 410 each, and 360
// with 16.
int norm_lines(int64_t rows, int64_t D) {
  const int64_t most = D <= 256 ? 1024 : D <= 8192 ? 512 : D <= 32768 ? 256 : 16;
  const int64_t few = std::min<int64_t>((rows + 3) / 4, 256);
  return (int)std::min(most, std::max({int64_t(1), few, rows / 16}));
}

hipError_t launch_layer_norm_fwd(const NormParams& p, int dtype, hipStream_t stream) {
  return dtype == 0 ? forward<float>(p, stream) : forward<__bf16>(p, stream);
}

hipError_t launch_layer_norm_bwd(const NormParams& p, float* dw, float* db, int dtype, hipStream_t stream) {
  return dtype == 0 ? backward<float>(p, dw, db, stream) : backward<__bf16>(p, dw, db, stream);
}

}  // namespace osm
