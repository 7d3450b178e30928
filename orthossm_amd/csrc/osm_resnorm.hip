// The residual norm on gfx950, forward and backward.
//
//   yh = N(y),  u = yh sigmoid(gate),  r = x + scale u,  rh = N(r),  n = rh w + b
//   N(v) = (v - m) s,  m = sum v / D (0 with rms),  s = 1 / sqrt(sum (v - m)^2 / D + eps)
//
//   g = w dn,  dr += s_r (g - mean(g) - rh mean(g rh)),  dx = dr
//   du = scale dr,  dgate = du yh sigmoid(gate) sigmoid(-gate),  e = du sigmoid(gate)
//   dy = s_y (e - mean(e) - yh mean(e yh))
//   dw = sum_rows dn rh,  db = sum_rows dn,  dscale = sum_rows dr u      (no mean(g), mean(e) with rms)
//
// What bounds both: the bytes of x, y, gate, r, n (x, y, gate, dr, dn, dx, dy, dgate);
// 262144 rows of 1024, blocks in bf16 around an fp32 stream: forward 640 us, 5.9 TB/s,
// backward 1230 us, 4.8 TB/s; all in bf16 449 and 897 us, 6.0 and 4.8 TB/s.
// A row is held in the registers of a quarter of a wave, of one, of four or of
// sixteen, so every input is read once, and the next row is on its way while one is
// worked on.  Not all registers fit where a thread holds 16 elements with an fp32 stream
// (rows of 513 to 1024 and 2049 to 4096) or 1024 threads hold a row: the backward then
// spills up to 97 of fp32 blocks (175 by 1024 threads) and 23 of bf16 ones (92), the
// forward by 1024 threads up to 80, and the rate falls (fp32, backward, 2^27 elements: rows of
// 512 834 us, 5.2 TB/s; of 1024 1318, 3.3; of 4096 1340, 3.2; of 8192 2108, 2.0).  The backward forms r again from x, y and gate and the saved statistics,
// unrounded as the forward had it; its workgroups walk rows a grid apart and keep
// their columns' sums in registers, each writes one line of them, and a second launch
// adds the lines in order, so the result does not depend on timing.
#include <algorithm>
#include <type_traits>

#include "osm_norm.h"
#include "osm_resnorm.h"
#include "osm_row.h"
#include "osm_wide_store.h"

// Fused multiply-adds are written where they are meant: e - mean(e) as one would
// leave the rounding of e in a gradient that is 0 (rows of one element).
#pragma clang fp contract(off)

namespace osm {
namespace {

// U elements of a row as loaded, in accesses of up to 16 bytes; past the row's end:
// zeros, and no stores.
template <typename T, int U>
struct Piece {
  static constexpr int kN = (int)sizeof(T) * U > 16 ? 16 / (int)sizeof(T) : U, kAccesses = U / kN;
  typedef T Vec __attribute__((ext_vector_type(kN)));
  typedef T Loose __attribute__((ext_vector_type(kN), aligned(sizeof(T))));
  Vec v[kAccesses];
  __device__ __forceinline__ void load(const T* p, int c, int D, bool vec) {
#pragma unroll
    for (int a = 0; a < kAccesses; ++a, c += kN) {
      Vec q = {};
      if (vec) {
        if (c < D) q = __builtin_nontemporal_load(reinterpret_cast<const Vec*>(p + c));
      } else if (c + kN <= D) {
        q = *reinterpret_cast<const Loose*>(p + c);
      } else {
#pragma unroll
        for (int i = 0; i < kN; ++i)
          if (c + i < D) q[i] = p[c + i];
      }
      v[a] = q;
    }
  }
  __device__ __forceinline__ float get(int i) const { return (float)v[i / kN][i % kN]; }
};

template <typename T, int U>
__device__ __forceinline__ void store_piece(T* p, const float (&f)[U], int c, int D, bool vec) {
  using P = Piece<T, U>;
#pragma unroll
  for (int a = 0; a < P::kAccesses; ++a, c += P::kN) {
    typename P::Vec q;
#pragma unroll
    for (int i = 0; i < P::kN; ++i) q[i] = (T)f[a * P::kN + i];
    if (vec) {
      if (c < D) {
        __builtin_nontemporal_store(q, reinterpret_cast<typename P::Vec*>(p + c));
        wide_store_wait();
      }
    } else if (c + P::kN <= D) {
      *reinterpret_cast<typename P::Loose*>(p + c) = q;
      wide_store_wait();
    } else {
#pragma unroll
      for (int i = 0; i < P::kN; ++i)
        if (c + i < D) p[c + i] = q[i];
    }
  }
}

// A row's statistics, in one store.
__device__ __forceinline__ void store_stats(float* p, float my, float sy, float mr, float sr) {
  typedef float Loose __attribute__((ext_vector_type(4), aligned(4)));
  *reinterpret_cast<Loose*>(p) = Loose{my, sy, mr, sr};
  wide_store_wait();
}

// Both off by |v| 2^-24 and a few units of 2^-24 (the hardware's reciprocal: the exact
// division takes twice the instructions of all the rest).
struct Gate {
  float o, rest;   // sigmoid(v), sigmoid(-v)
};
__device__ __forceinline__ Gate gate_of(float v) {
  const float e = __builtin_amdgcn_exp2f(-1.44269504f * __builtin_fabsf(v)), r = __builtin_amdgcn_rcpf(1.0f + e), s = e * r;
  return v >= 0.0f ? Gate{r, s} : Gate{s, r};
}

template <int TPR>
struct RowThreads {
  static constexpr int kThreads = TPR > 256 ? TPR : 256, kRows = kThreads / TPR;
};

// (v - mean) / spread of a row in registers, zeros past its end; the sums alternate
// between red's halves.
template <int TPR, int NV, int U>
__device__ __forceinline__ void normalise(float (&v)[NV][U], int D, int u, float eps, bool rms, float (*red)[16][1], int& par,
                                          float& mean, float& rs) {
  float s[1] = {0.0f};
  mean = 0.0f;
  if (!rms) {
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < U; ++i) s[0] += v[k][i];
    row_sum<TPR>(s, red[par]);
    par ^= 1;
    mean = s[0] / (float)D;
    s[0] = 0.0f;
  }
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < U; ++i) {
      v[k][i] = (u + k * TPR) * U + i < D ? v[k][i] - mean : 0.0f;
      s[0] = __builtin_fmaf(v[k][i], v[k][i], s[0]);
    }
  row_sum<TPR>(s, red[par]);
  par ^= 1;
  rs = 1.0f / sqrtf(s[0] / (float)D + eps);
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < U; ++i) v[k][i] *= rs;
}

// COUNT fp32 parameters of a row's columns, in LDS while that leaves room for two
// workgroups a CU (rows up to 4096), else in registers; `fill` where there are none, zeros
// past the row's end.
template <int TPR, int NV, int U, int COUNT>
struct Params {
  static constexpr int kCols = TPR * NV * U;
  static constexpr bool kShared = kCols <= 4096;
  typedef float Four __attribute__((ext_vector_type(4)));
  float own[kShared ? 1 : COUNT][NV][U];
  float* lds;
  int u;
  static constexpr int kLds = kShared ? COUNT * kCols : 1;
  __device__ __forceinline__ Params(float* s, int thread) : lds(s), u(thread) {}
  __device__ __forceinline__ void set(int which, const float* w, float fill, int D) {
    if constexpr (kShared) {
      for (int c = threadIdx.x; c < kCols; c += blockDim.x) lds[which * kCols + c] = c < D ? (w ? w[c] : fill) : 0.0f;
    } else {
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < U; ++i) {
          const int c = (u + k * TPR) * U + i;
          own[which][k][i] = c < D ? (w ? w[c] : fill) : 0.0f;
        }
    }
  }
  __device__ __forceinline__ void get(int which, int k, float (&v)[U]) const {
    if constexpr (kShared) {
#pragma unroll
      for (int i = 0; i < U; i += 4) {
        const Four f = *reinterpret_cast<const Four*>(lds + which * kCols + (u + k * TPR) * U + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[i + j] = f[j];
      }
    } else {
#pragma unroll
      for (int i = 0; i < U; ++i) v[i] = own[which][k][i];
    }
  }
};

// TX: the residual stream's type, TY: the block's; TPR threads a row, max(TPR, 256)
// a workgroup, units of U columns.
template <typename TX, typename TY, int U, int TPR, int NV>
__global__ void __launch_bounds__(RowThreads<TPR>::kThreads) resnorm_fwd_kernel(const ResnormParams p) {
  constexpr int kRows = RowThreads<TPR>::kRows;
  __shared__ float red[2][16][1];
  using P = Params<TPR, NV, U, 3>;
  __shared__ __attribute__((aligned(16))) float shared[P::kLds];
  const int u = threadIdx.x % TPR, D = (int)p.D;
  const int64_t step = (int64_t)gridDim.x * kRows;
  int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / TPR;
  int half = 0;
  Piece<TX, U> rx[NV];
  Piece<TY, U> ry[NV], rg[NV];
  auto fetch = [&](int64_t at) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (u + k * TPR) * U;
      ry[k].load(static_cast<const TY*>(p.y) + at * p.y_s, c, D, p.vec);
      if (p.gate) rg[k].load(static_cast<const TY*>(p.gate) + at * p.gate_s, c, D, p.vec);
      rx[k].load(static_cast<const TX*>(p.x) + at * p.x_s, c, D, p.vec);
    }
  };
  if (row < p.rows) fetch(row);
  P par(shared, u);
  par.set(0, p.weight, 1.0f, D);
  par.set(1, p.bias, 0.0f, D);
  par.set(2, p.scale, 1.0f, D);
  __syncthreads();
  // (every thread of a workgroup runs the same trips: kRows is 1 where row_sum has barriers)
  for (; row < p.rows; row += step) {
    float x[NV][U], y[NV][U], o[NV][U];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      par.get(2, k, o[k]);
#pragma unroll
      for (int i = 0; i < U; ++i) {
        x[k][i] = rx[k].get(i);
        y[k][i] = ry[k].get(i);
        if (p.gate) o[k][i] *= gate_of(rg[k].get(i)).o;
      }
    }
    if (row + step < p.rows) fetch(row + step);
    float my = 0.0f, sy = 1.0f, mr, sr;
    if (p.norm_y) normalise<TPR>(y, D, u, p.eps, p.rms, red, half, my, sy);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
      for (int i = 0; i < U; ++i) x[k][i] = __builtin_fmaf(o[k][i], y[k][i], x[k][i]);
      store_piece<TX, U>(static_cast<TX*>(p.r) + row * p.r_s, x[k], (u + k * TPR) * U, D, p.vec);
    }
    normalise<TPR>(x, D, u, p.eps, p.rms, red, half, mr, sr);
    if (p.stats && u == 0) store_stats(p.stats + 4 * row, my, sy, mr, sr);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float w[U], b[U];
      par.get(0, k, w);
      par.get(1, k, b);
#pragma unroll
      for (int i = 0; i < U; ++i) x[k][i] = __builtin_fmaf(x[k][i], w[i], b[i]);
      store_piece<TY, U>(static_cast<TY*>(p.n) + row * p.n_s, x[k], (u + k * TPR) * U, D, p.vec);
    }
  }
}

template <typename TX, typename TY, int U, int TPR, int NV>
__global__ void __launch_bounds__(RowThreads<TPR>::kThreads, 2) resnorm_bwd_kernel(const ResnormParams p) {
  constexpr int kRows = RowThreads<TPR>::kRows;
  using P = Params<TPR, NV, U, 2>;
  __shared__ float red[2][16][2];
  __shared__ __attribute__((aligned(16))) float shared[P::kLds];
  const int u = threadIdx.x % TPR, D = (int)p.D;
  float dw[NV][U], db[NV][U], ds[NV][U];
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < U; ++i) dw[k][i] = db[k][i] = ds[k][i] = 0.0f;
  const int64_t step = (int64_t)gridDim.x * kRows;
  int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / TPR;
  int half = 0;
  Piece<TX, U> next_x[NV], next_r[NV] = {};
  Piece<TY, U> next_y[NV], next_g[NV] = {}, next_n[NV] = {};
  float st[4];
  auto fetch = [&](int64_t at) {
#pragma unroll
    for (int i = 0; i < 4; ++i) st[i] = p.stats[4 * at + i];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (u + k * TPR) * U;
      next_y[k].load(static_cast<const TY*>(p.y) + at * p.y_s, c, D, p.vec);
      if (p.gate) next_g[k].load(static_cast<const TY*>(p.gate) + at * p.gate_s, c, D, p.vec);
      next_x[k].load(static_cast<const TX*>(p.x) + at * p.x_s, c, D, p.vec);
      if (p.gn) next_n[k].load(static_cast<const TY*>(p.gn) + at * p.gn_s, c, D, p.vec);
      if (p.gr) next_r[k].load(static_cast<const TX*>(p.gr) + at * p.gr_s, c, D, p.vec);
    }
  };
  if (row < p.rows) fetch(row);
  P par(shared, u);
  par.set(0, p.weight, 1.0f, D);
  par.set(1, p.scale, 1.0f, D);
  __syncthreads();
  for (; row < p.rows; row += step) {
    // What the second pass takes again stays as it was loaded: its values are formed twice,
    // in fewer registers.
    Piece<TY, U> y[NV], gate[NV], n[NV];
    Piece<TX, U> gr[NV];
    float rh[NV][U], dr[NV][U];
    const float sy = st[1], sr = st[3], my = st[0], mr = st[2];
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      y[k] = next_y[k];
      gate[k] = next_g[k];
      n[k] = next_n[k];
      gr[k] = next_r[k];
      float w[U], sc[U];
      par.get(0, k, w);
      par.get(1, k, sc);
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const float o = p.gate ? gate_of(gate[k].get(i)).o : 1.0f, dn = n[k].get(i);
        // (the forward's r, to the last bit)
        const float r = __builtin_fmaf(sc[i] * o, (y[k].get(i) - my) * sy, next_x[k].get(i));
        rh[k][i] = (r - mr) * sr;
        dw[k][i] = __builtin_fmaf(dn, rh[k][i], dw[k][i]);
        db[k][i] += dn;
        const float g = dn * w[i];       // zeros past the row's end: dn and w are
        s[0] += g;
        s[1] = __builtin_fmaf(g, rh[k][i], s[1]);
      }
    }
    if (row + step < p.rows) fetch(row + step);
    row_sum<TPR>(s, red[half]);
    half ^= 1;
    float a = p.rms ? 0.0f : s[0] / (float)D, c = s[1] / (float)D;
    s[0] = s[1] = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float w[U], sc[U], dg[U];
      par.get(0, k, w);
      par.get(1, k, sc);
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const Gate q = p.gate ? gate_of(gate[k].get(i)) : Gate{1.0f, 0.0f};
        const float yh = (y[k].get(i) - my) * sy;
        dr[k][i] = gr[k].get(i) + sr * (n[k].get(i) * w[i] - a - rh[k][i] * c);
        ds[k][i] = __builtin_fmaf(dr[k][i], yh * q.o, ds[k][i]);
        const float e = dr[k][i] * sc[i] * q.o;   // zero past the row's end: sc is
        dg[i] = q.rest * (e * yh);
        s[0] += e;
        s[1] = __builtin_fmaf(e, yh, s[1]);
        rh[k][i] = e;
      }
      const int at = (u + k * TPR) * U;
      if (p.gx) store_piece<TX, U>(static_cast<TX*>(p.gx) + row * p.gx_s, dr[k], at, D, p.vec);
      if (p.gg) store_piece<TY, U>(static_cast<TY*>(p.gg) + row * p.gg_s, dg, at, D, p.vec);
    }
    a = c = 0.0f;
    if (p.norm_y) {
      row_sum<TPR>(s, red[half]);
      half ^= 1;
      a = p.rms ? 0.0f : s[0] / (float)D;
      c = s[1] / (float)D;
    }
    if (p.gy)
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        float dy[U];
#pragma unroll
        for (int i = 0; i < U; ++i) dy[i] = sy * (rh[k][i] - a - (y[k].get(i) - my) * sy * c);
        store_piece<TY, U>(static_cast<TY*>(p.gy) + row * p.gy_s, dy, (u + k * TPR) * U, D, p.vec);
      }
  }
  // This workgroup's line of sums: its row groups in order.
  float* const line = p.part + (int64_t)blockIdx.x * 3 * D;
  if constexpr (kRows > 1) {
    __shared__ float sums[kRows - 1][3][TPR * U];
    const int group = threadIdx.x / TPR;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      __syncthreads();
      if (group > 0)
#pragma unroll
        for (int i = 0; i < U; ++i) {
          sums[group - 1][0][i * TPR + u] = dw[k][i];
          sums[group - 1][1][i * TPR + u] = db[k][i];
          sums[group - 1][2][i * TPR + u] = ds[k][i];
        }
      __syncthreads();
      if (group == 0)
#pragma unroll 3
        for (int q = 0; q < kRows - 1; ++q)
#pragma unroll
          for (int i = 0; i < U; ++i) {
            dw[k][i] += sums[q][0][i * TPR + u];
            db[k][i] += sums[q][1][i * TPR + u];
            ds[k][i] += sums[q][2][i * TPR + u];
          }
    }
    if (group > 0) return;
  }
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int c = (u + k * TPR) * U + i;
      if (c < D) {
        line[c] = dw[k][i];
        line[D + c] = db[k][i];
        line[2 * (int64_t)D + c] = ds[k][i];
      }
    }
}

constexpr int kLongThreads = 1024;

// An element of long rows, formed again wherever it is needed.
template <typename TX, typename TY>
struct LongRow {
  const TX* x;
  const TY *y, *gate;
  const ResnormParams& p;
  __device__ LongRow(const ResnormParams& q, int64_t row) : p(q) {
    x = static_cast<const TX*>(p.x) + row * p.x_s;
    y = static_cast<const TY*>(p.y) + row * p.y_s;
    gate = p.gate ? static_cast<const TY*>(p.gate) + row * p.gate_s : nullptr;
  }
  __device__ __forceinline__ float scale(int64_t c) const { return p.scale ? p.scale[c] : 1.0f; }
  __device__ __forceinline__ Gate open(int64_t c) const { return gate ? gate_of((float)gate[c]) : Gate{1.0f, 0.0f}; }
  __device__ __forceinline__ float yh(int64_t c, float m, float s) const { return ((float)y[c] - m) * s; }
  __device__ __forceinline__ float r(int64_t c, float m, float s) const {
    return __builtin_fmaf(scale(c) * open(c).o, yh(c, m, s), (float)x[c]);
  }
};

// Mean and 1 / spread of f(0) .. f(D - 1).
template <typename F>
__device__ __forceinline__ void long_stats(const ResnormParams& p, F f, float (*red)[16][1], int& par, float& mean, float& rs) {
  float s[1] = {0.0f};
  mean = 0.0f;
  if (!p.rms) {
    for (int64_t c = threadIdx.x; c < p.D; c += kLongThreads) s[0] += f(c);
    row_sum<kLongThreads>(s, red[par]);
    par ^= 1;
    mean = s[0] / (float)p.D;
    s[0] = 0.0f;
  }
  for (int64_t c = threadIdx.x; c < p.D; c += kLongThreads) {
    const float d = f(c) - mean;
    s[0] = __builtin_fmaf(d, d, s[0]);
  }
  row_sum<kLongThreads>(s, red[par]);
  par ^= 1;
  rs = 1.0f / sqrtf(s[0] / (float)p.D + p.eps);
}

// Rows too long for registers: a workgroup a row, read again for every sum.
template <typename TX, typename TY>
__global__ void __launch_bounds__(kLongThreads) resnorm_fwd_long_kernel(const ResnormParams p) {
  __shared__ float red[2][16][1];
  int par = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const LongRow<TX, TY> q(p, row);
    float my = 0.0f, sy = 1.0f, mr, sr;
    if (p.norm_y) long_stats(p, [&](int64_t c) { return (float)q.y[c]; }, red, par, my, sy);
    long_stats(p, [&](int64_t c) { return q.r(c, my, sy); }, red, par, mr, sr);
    if (p.stats && threadIdx.x == 0) store_stats(p.stats + 4 * row, my, sy, mr, sr);
    for (int64_t c = threadIdx.x; c < p.D; c += kLongThreads) {
      const float r = q.r(c, my, sy);
      static_cast<TX*>(p.r)[row * p.r_s + c] = (TX)r;
      static_cast<TY*>(p.n)[row * p.n_s + c] =
          (TY)__builtin_fmaf((r - mr) * sr, p.weight ? p.weight[c] : 1.0f, p.bias ? p.bias[c] : 0.0f);
    }
  }
}

// dr of an element of a long row, whose sums of g and g rh (over D) are a and c0.
template <typename TX, typename TY>
__device__ __forceinline__ float long_dr(const ResnormParams& p, int64_t row, int64_t c, float rh, float sr, float a, float c0) {
  const float dn = p.gn ? (float)static_cast<const TY*>(p.gn)[row * p.gn_s + c] : 0.0f;
  const float gr = p.gr ? (float)static_cast<const TX*>(p.gr)[row * p.gr_s + c] : 0.0f;
  return gr + sr * (dn * (p.weight ? p.weight[c] : 1.0f) - a - rh * c0);
}

template <typename TX, typename TY>
__global__ void __launch_bounds__(kLongThreads) resnorm_bwd_long_kernel(const ResnormParams p) {
  __shared__ float red[2][16][2];
  int par = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const LongRow<TX, TY> q(p, row);
    const float my = p.stats[4 * row], sy = p.stats[4 * row + 1], mr = p.stats[4 * row + 2], sr = p.stats[4 * row + 3];
    float s[2] = {0.0f, 0.0f};
    if (p.gn)
      for (int64_t c = threadIdx.x; c < p.D; c += kLongThreads) {
        const float g = (float)static_cast<const TY*>(p.gn)[row * p.gn_s + c] * (p.weight ? p.weight[c] : 1.0f);
        s[0] += g;
        s[1] = __builtin_fmaf(g, (q.r(c, my, sy) - mr) * sr, s[1]);
      }
    row_sum<kLongThreads>(s, red[par]);
    par ^= 1;
    const float a = p.rms ? 0.0f : s[0] / (float)p.D, c0 = s[1] / (float)p.D;
    if (threadIdx.x == 0) {
      p.sums[2 * row] = a;
      p.sums[2 * row + 1] = c0;
    }
    float a2 = 0.0f, c2 = 0.0f;
    if (p.norm_y) {
      s[0] = s[1] = 0.0f;
      for (int64_t c = threadIdx.x; c < p.D; c += kLongThreads) {
        const float e = long_dr<TX, TY>(p, row, c, (q.r(c, my, sy) - mr) * sr, sr, a, c0) * q.scale(c) * q.open(c).o;
        s[0] += e;
        s[1] = __builtin_fmaf(e, q.yh(c, my, sy), s[1]);
      }
      row_sum<kLongThreads>(s, red[par]);
      par ^= 1;
      a2 = p.rms ? 0.0f : s[0] / (float)p.D;
      c2 = s[1] / (float)p.D;
    }
    for (int64_t c = threadIdx.x; c < p.D; c += kLongThreads) {
      const float yh = q.yh(c, my, sy), dr = long_dr<TX, TY>(p, row, c, (q.r(c, my, sy) - mr) * sr, sr, a, c0);
      const Gate o = q.open(c);
      const float e = dr * q.scale(c) * o.o;
      if (p.gx) static_cast<TX*>(p.gx)[row * p.gx_s + c] = (TX)dr;
      if (p.gg) static_cast<TY*>(p.gg)[row * p.gg_s + c] = (TY)(o.rest * (e * yh));
      if (p.gy) static_cast<TY*>(p.gy)[row * p.gy_s + c] = (TY)(sy * (e - a2 - yh * c2));
    }
  }
}

// A line of sums of long rows: workgroup (columns, line) takes rows line, line + lines, ..
template <typename TX, typename TY>
__global__ void __launch_bounds__(256) resnorm_columns_kernel(const ResnormParams p) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= p.D) return;
  float dw = 0.0f, db = 0.0f, ds = 0.0f;
  for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
    const LongRow<TX, TY> q(p, row);
    const float my = p.stats[4 * row], sy = p.stats[4 * row + 1], mr = p.stats[4 * row + 2], sr = p.stats[4 * row + 3];
    const float rh = (q.r(c, my, sy) - mr) * sr;
    const float dn = p.gn ? (float)static_cast<const TY*>(p.gn)[row * p.gn_s + c] : 0.0f;
    dw = __builtin_fmaf(dn, rh, dw);
    db += dn;
    ds = __builtin_fmaf(long_dr<TX, TY>(p, row, c, rh, sr, p.sums[2 * row], p.sums[2 * row + 1]),
                        q.yh(c, my, sy) * q.open(c).o, ds);
  }
  float* const line = p.part + (int64_t)blockIdx.y * 3 * p.D;
  line[c] = dw;
  line[p.D + c] = db;
  line[2 * p.D + c] = ds;
}

constexpr int kFoldCols = 32, kFoldGroups = 32;

// The parameters' gradients from the lines, 32 columns a workgroup: group g adds lines
// g, g + 32, ..; then the groups in order.
__global__ void __launch_bounds__(kFoldCols * kFoldGroups) resnorm_fold_kernel(const float* part, float* dw, float* db, float* ds,
                                                                               int64_t D, int lines) {
  __shared__ float red[kFoldGroups][kFoldCols];
  const int cl = threadIdx.x % kFoldCols, g = threadIdx.x / kFoldCols;
  const int64_t c = (int64_t)blockIdx.x * kFoldCols + cl;
  float s = 0.0f;
  if (c < 3 * D) {
#pragma unroll 8
    for (int i = g; i < lines; i += kFoldGroups) s += part[(int64_t)i * 3 * D + c];
  }
  red[g][cl] = s;
  __syncthreads();
  if (g == 0 && c < 3 * D) {
#pragma unroll
    for (int q = 1; q < kFoldGroups; ++q) s += red[q][cl];
    float* const dst = c < D ? dw : c < 2 * D ? db : ds;
    if (dst) dst[c % D] = s;
  }
}

// Calls go(TPR, NV) for the fewest threads that hold a row, up to 16 elements each
// (LAST in the case of 1024 threads), or long_rows() past that.  (Rows of 1024 columns around
// an fp32 stream by 256 threads in place of 64: forward 841 us for 660, backward the same.)
template <int U, int LAST, typename Go, typename Long>
void by_length(int64_t D, Go go, Long long_rows) {
  const int64_t units = (D + U - 1) / U;
  auto pick = [&](auto tpr) {
    constexpr int TPR = decltype(tpr)::value, most = TPR == 16 ? 1 : (TPR == 1024 ? LAST : 16) / U;
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

// Workgroups of a forward, each of which walks rows a grid apart (262144 rows of 1024 around an
// fp32 stream: 2048, 8192 and 32768 take 678, 660 and 643 us).
constexpr int kMaxGroups = 32768;
constexpr int kLastFwd = 16, kLastBwd = 8;   // elements of a thread where 1024 hold a row

// Columns of a unit: 16 bytes of the wider type, so that a wave's accesses to either are
// without gaps (8 columns of an fp32 stream: 871 and 1368 us for 660 and 1317).
template <typename TX>
constexpr int kUnit = 16 / (int)sizeof(TX);

template <typename TX, typename TY>
hipError_t forward(const ResnormParams& p, hipStream_t stream) {
  constexpr int U = kUnit<TX>;
  by_length<U, kLastFwd>(
      p.D,
      [&](auto tpr, auto nv) {
        constexpr int TPR = decltype(tpr)::value, NV = decltype(nv)::value;
        const int64_t groups = (p.rows + RowThreads<TPR>::kRows - 1) / RowThreads<TPR>::kRows;
        hipLaunchKernelGGL((resnorm_fwd_kernel<TX, TY, U, TPR, NV>), dim3((unsigned)std::min<int64_t>(groups, kMaxGroups)),
                           dim3(RowThreads<TPR>::kThreads), 0, stream, p);
      },
      [&] {
        hipLaunchKernelGGL((resnorm_fwd_long_kernel<TX, TY>), dim3((unsigned)std::min<int64_t>(p.rows, kMaxGroups)),
                           dim3(kLongThreads), 0, stream, p);
      });
  return hipGetLastError();
}

template <typename TX, typename TY>
hipError_t backward(const ResnormParams& p, float* dw, float* db, float* ds, hipStream_t stream) {
  constexpr int U = kUnit<TX>;
  const int lines = norm_lines(p.rows, p.D);
  hipError_t e = hipSuccess;
  by_length<U, kLastBwd>(
      p.D,
      [&](auto tpr, auto nv) {
        constexpr int TPR = decltype(tpr)::value, NV = decltype(nv)::value;
        hipLaunchKernelGGL((resnorm_bwd_kernel<TX, TY, U, TPR, NV>), dim3(lines), dim3(RowThreads<TPR>::kThreads), 0, stream, p);
      },
      [&] {
        hipLaunchKernelGGL((resnorm_bwd_long_kernel<TX, TY>), dim3((unsigned)std::min<int64_t>(p.rows, kMaxGroups)),
                           dim3(kLongThreads), 0, stream, p);
        e = hipGetLastError();
        if (e == hipSuccess)
          hipLaunchKernelGGL((resnorm_columns_kernel<TX, TY>), dim3((unsigned)((p.D + 255) / 256), lines), dim3(256), 0, stream, p);
      });
  if (e == hipSuccess) e = hipGetLastError();
  if (e != hipSuccess || (!dw && !db && !ds)) return e;
  hipLaunchKernelGGL(resnorm_fold_kernel, dim3((unsigned)((3 * p.D + kFoldCols - 1) / kFoldCols)), dim3(kFoldCols * kFoldGroups), 0,
                     stream, p.part, dw, db, ds, p.D, lines);
  return hipGetLastError();
}

// f(TX{}, TY{}) for the types of the stream and the block.
template <typename F>
hipError_t by_types(int stream_dtype, int block_dtype, F f) {
  if (block_dtype == 0) return f(0.0f, 0.0f);
  return stream_dtype == 0 ? f(0.0f, (__bf16)0.0f) : f((__bf16)0.0f, (__bf16)0.0f);
}

}  // namespace

bool resnorm_long(int64_t D) { return D > 1024 * kLastBwd; }

hipError_t launch_resnorm_fwd(const ResnormParams& p, int stream_dtype, int block_dtype, hipStream_t stream) {
  return by_types(stream_dtype, block_dtype, [&](auto tx, auto ty) { return forward<decltype(tx), decltype(ty)>(p, stream); });
}

hipError_t launch_resnorm_bwd(const ResnormParams& p, float* dw, float* db, float* ds, int stream_dtype, int block_dtype,
                              hipStream_t stream) {
  return by_types(stream_dtype, block_dtype,
                  [&](auto tx, auto ty) { return backward<decltype(tx), decltype(ty)>(p, dw, db, ds, stream); });
}

}  // namespace osm
