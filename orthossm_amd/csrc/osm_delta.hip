// The gated delta rule on gfx950: chunked forward.
//
//   S_t = e^{g_t} S_{t-1} + k_t u_t^T,   u_t = beta_t (v_t - e^{g_t} S_{t-1}^T k_t),   o_t = scale S_t^T q_t
//
// Over a chunk of 64 tokens with start state S, G = the running sum of g,
// M_ij = e^{G_i - G_j} (i >= j), L = M o K K^T below the diagonal and
// P = M o Q K^T on and below it, the updates solve a triangular system.  With
//   Z = L (I + diag(beta) L)^-1    (zero on and above the diagonal)
// its two inverses are (I + L diag(beta))^-1 = I - Z diag(beta) and
// (I + diag(beta) L)^-1 = I - diag(beta) Z, without dividing by beta, so
//   X = V - e^G K S,  Y = X - Z (beta X),  U = beta Y,  O = scale (e^G Q S + P U)
// and the chunk's end state is affine in S, with Kt = e^{G_last - G} K:
//   S' = A S + B,   A = e^{G_last} I - Kt^T W,   W = beta (e^G K - Z (beta e^G K))
//                   B = Kt^T beta (V - Z (beta V))
//
// Three launches: `prepare` forms Z, A and B of every chunk at once, `scan`
// walks the chunks of a row with one product each (its 16 columns of S stay in
// the waves' accumulators), writing every chunk's start state over its B, and
// `output` forms O of every chunk at once.  All products run on the fp32 matrix
// instruction: the states and the gates' gradients are fp32 results.
#include <type_traits>

#include "osm_delta.h"

namespace osm {
namespace {

using namespace delta;

constexpr int kThreads = 256;

// Z from L in place (tile zs, L strictly lower, zeros elsewhere): the four
// diagonal 16x16 blocks by substitution, row i from the rows before it (Z_i =
// L_i - sum_j L_ij beta_j Z_j), then block pairs: for L = [[a, 0], [c, d]],
// Z_c = (I - Z_d beta) (L_c - L_c beta Z_a), the 16-wide ones, then the 32-wide.
__device__ void invert(float* zs, const Gates& gt) {
  const int wave = threadIdx.x >> 6, l = threadIdx.x & 63;
  if (wave == 0) {
    const int c = l & 15, o = 16 * (l >> 4);
    float* const base = zs + o * kLd + o;
    float z[16], bz[16];   // column c of the block's Z, and beta Z
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float v = base[i * kLd + c];
#pragma unroll
      for (int j = 0; j < i; ++j) v = __builtin_fmaf(-base[i * kLd + j], bz[j], v);
      z[i] = v;
      bz[i] = gt.beta[o + i] * v;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // every lane has read its rows
#pragma unroll
    for (int i = 0; i < 16; ++i) base[i * kLd + c] = z[i];
  }
  __syncthreads();
  // 16-wide: waves 0 and 1 take the pairs (0, 1) and (2, 3).
  {
    const int a = 32 * (wave & 1), d = a + 16;
    f32x4 acc[1], q[1];
    if (wave < 2) {
      clear(acc);
      mma<1, false, false, true>(acc, zs, d, zs, a, a, d, gt.beta);   // L_c beta Z_a
      get(q, zs, d, a);
      q[0] -= acc[0];
    }
    __syncthreads();
    if (wave < 2) put(zs, q, d, a);
    __syncthreads();
    if (wave < 2) {
      clear(acc);
      mma<1, false, false, true>(acc, zs, d, zs, a, d, d + 16, gt.beta);   // Z_d beta (..)
      q[0] -= acc[0];
    }
    __syncthreads();
    if (wave < 2) put(zs, q, d, a);
    __syncthreads();
  }
  // 32-wide: a 16x16 tile a wave.
  {
    const int r0 = 32 + 16 * (wave >> 1), c0 = 16 * (wave & 1);
    f32x4 acc[1], q[1];
    clear(acc);
    mma<1, false, false, true>(acc, zs, r0, zs, c0, 0, 32, gt.beta);
    get(q, zs, r0, c0);
    q[0] -= acc[0];
    __syncthreads();
    put(zs, q, r0, c0);
    __syncthreads();
    clear(acc);
    mma<1, false, false, true>(acc, zs, r0, zs, c0, 32, 64, gt.beta);
    q[0] -= acc[0];
    __syncthreads();
    put(zs, q, r0, c0);
    __syncthreads();
  }
}

// Z, A and B of a chunk.  LDS: three tiles (52 KB), so that three workgroups
// share a CU; head sizes above 64 go by blocks of 64 columns.
template <typename T>
__global__ void __launch_bounds__(kThreads) delta_prepare_kernel(const DeltaParams p) {
  __shared__ __attribute__((aligned(16))) float zs[kTile], ks[kTile], ws[kTile];
  __shared__ __attribute__((aligned(16))) Gates gt;
  const At w = chunk_at(p, blockIdx.x);
  if (w.rows == 0) return;
  const int r0 = 16 * (threadIdx.x >> 6), hk = w.h / (p.H / p.Hk);
  load_gates(&gt, p.g, p.beta, w.b, w.t0, w.h, w.rows);
  const T* const k = row_ptr<T>(p.k, w.b, w.t0, hk);
  const T* const v = row_ptr<T>(p.v, w.b, w.t0, w.h);
  const bool vec = p.vec;
  f32x4 acc[4];
  clear(acc);
  for (int kb = 0; kb < p.dkp; kb += 64) {
    const int kw = min(64, p.dkp - kb);
    if (kb) __syncthreads();
    load_tile<kThreads>(ks, k + kb, p.k.ss, w.rows, p.dk_ - kb, kw, vec);
    __syncthreads();
    mma<4, false, true>(acc, ks, r0, ks, 0, 0, kw);
  }
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = out_row(r0, i), col = out_col(0, c);
      acc[c][i] = row > col ? acc[c][i] * decay_between(gt, row, col) : 0.0f;
    }
  put(zs, acc, r0, 0);
  __syncthreads();
  invert(zs, gt);
  const int64_t chunk = blockIdx.x;
  float* const zg = p.z + chunk * 4096;
  for (int e = threadIdx.x; e < 1024; e += kThreads)
    *reinterpret_cast<f32x4*>(zg + 4 * e) = *reinterpret_cast<const f32x4*>(zs + (e >> 4) * kLd + 4 * (e & 15));
  const int nkb = (p.dkp + 63) / 64;
  int held = nkb - 1;   // the block of K in ks
  auto hold = [&](int blk) {
    if (blk == held) return;
    __syncthreads();
    load_tile<kThreads>(ks, k + 64 * blk, p.k.ss, w.rows, p.dk_ - 64 * blk, min(64, p.dkp - 64 * blk), vec);
    held = blk;
    __syncthreads();
  };
  // A by blocks of columns
  float* const ag = p.a + chunk * p.dkp * p.dkp;
  for (int cb = 0; cb < nkb; ++cb) {
    const int cw = min(64, p.dkp - 64 * cb);
    hold(cb);
    clear(acc);
    mma<4, false, false, true>(acc, zs, r0, ks, 0, 0, r0 + 16, gt.bgam);
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = out_row(r0, i), col = out_col(0, c);
        acc[c][i] = gt.end[row] * gt.beta[row] * (gt.gam[row] * (col < cw ? ks[row * kLd + col] : 0.0f) - acc[c][i]);
      }
    __syncthreads();   // the previous block's product has read ws
    put(ws, acc, r0, 0);
    __syncthreads();
    for (int rb = 0; rb < nkb; ++rb) {
      const int rw = min(64, p.dkp - 64 * rb);
      hold(rb);
      if (r0 >= rw) continue;   // (hold's barriers are behind every wave)
      clear(acc);
      mma<4, true, false>(acc, ks, r0, ws, 0, 0, 64);
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = 64 * rb + out_row(r0, i), col = out_col(0, c);
          if (col < cw) ag[(int64_t)row * p.dkp + 64 * cb + col] = (row == 64 * cb + col ? gt.last : 0.0f) - acc[c][i];
        }
    }
  }
  // B by blocks of columns
  float* const sg = p.s + chunk * p.dkp * p.dvp;
  for (int vb = 0; vb < p.dvp; vb += 64) {
    const int vw = min(64, p.dvp - vb);
    __syncthreads();
    load_tile<kThreads>(ws, v + vb, p.v.ss, w.rows, p.dv_ - vb, 64, vec);
    __syncthreads();
    clear(acc);
    mma<4, false, false, true>(acc, zs, r0, ws, 0, 0, r0 + 16, gt.beta);
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = out_row(r0, i);
        acc[c][i] = gt.end[row] * gt.beta[row] * (ws[row * kLd + out_col(0, c)] - acc[c][i]);
      }
    __syncthreads();
    put(ws, acc, r0, 0);
    __syncthreads();
    for (int rb = 0; rb < nkb; ++rb) {
      const int rw = min(64, p.dkp - 64 * rb);
      hold(rb);
      if (r0 >= rw) continue;
      clear(acc);
      mma<4, true, false>(acc, ks, r0, ws, 0, 0, 64);
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int col = out_col(0, c);
          if (col < vw) sg[(int64_t)(64 * rb + out_row(r0, i)) * p.dvp + vb + col] = acc[c][i];
        }
    }
  }
}

// S' = A S + B over the chunks of a row, in order or in reverse, for 16 columns
// of S: wave w holds rows 16 w .. 16 w + 15 of S and of A, and S passes between
// the waves through LDS, transposed ([column][row], so that both the
// accumulators' four rows and the product's four terms are one 16-byte access),
// in two buffers: one barrier a chunk.  x holds B and receives the state before
// the chunk.  KT = dkp / 16.
//
// What bounds it: the chain of chunks, each KT dependent-in-pairs matrix
// instructions of 4 KT .. plus the exchange.
template <int KT>
__global__ void __launch_bounds__(64 * KT) delta_scan_kernel(const float* a, float* x, const float* init, float* fin,
                                                             const int* lengths, int S, int N, int BH, int H, int dk,
                                                             int dv, int dvp, bool reverse) {
  constexpr int kDkp = 16 * KT, kRow = kDkp + 4;
  __shared__ __attribute__((aligned(16))) float st[2][16 * kRow];
  // The column slices of a head share A, so they take one XCD (workgroups go
  // round the eight XCDs by their index).
  const int ns = dvp / kDeltaSlice, j = blockIdx.x >> 3, bh = (j / ns) * 8 + (blockIdx.x & 7);
  if (bh >= BH) return;
  const int wave = threadIdx.x >> 6, l = threadIdx.x & 63, r = l & 15, g = l >> 4;
  const int col = kDeltaSlice * (j % ns) + r, row = 16 * wave + 4 * g;
  const int tokens = lengths ? min(max(lengths[bh / H], 0), S) : S;
  const int n = (tokens + kDeltaChunk - 1) / kDeltaChunk;
  a += (int64_t)bh * N * kDkp * kDkp + (int64_t)(16 * wave + r) * kDkp + 4 * g;
  x += (int64_t)bh * N * kDkp * dvp + (int64_t)row * dvp + col;
  const int64_t io = (int64_t)bh * dk * dv + (int64_t)row * dv + col;
  f32x4 s = zero4();
  if (init)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (row + i < dk && col < dv) s[i] = init[io + (int64_t)i * dv];
  auto at = [&](int c) { return (int64_t)(reverse ? n - 1 - c : c); };
  f32x4 an[KT], bn;
  auto fetch = [&](int c) {
    const float* const ap = a + at(c) * kDkp * kDkp;
    const float* const xp = x + at(c) * kDkp * dvp;
#pragma unroll
    for (int k = 0; k < KT; ++k) an[k] = load4(ap + 16 * k);
#pragma unroll
    for (int i = 0; i < 4; ++i) bn[i] = xp[(int64_t)i * dvp];
  };
  if (n > 0) fetch(0);
  for (int c = 0; c < n; ++c) {
    float* const buf = st[c & 1];
    *reinterpret_cast<f32x4*>(buf + r * kRow + row) = s;
    f32x4 ac[KT], acc0 = bn, acc1 = zero4();
#pragma unroll
    for (int k = 0; k < KT; ++k) ac[k] = an[k];
    float* const xp = x + at(c) * kDkp * dvp;
    if (c + 1 < n) fetch(c + 1);
#pragma unroll
    for (int i = 0; i < 4; ++i) xp[(int64_t)i * dvp] = s[i];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < KT; ++k) {
      const f32x4 b = *reinterpret_cast<const f32x4*>(buf + r * kRow + 16 * k + 4 * g);
      acc0 = __builtin_amdgcn_mfma_f32_16x16x4f32(ac[k][0], b[0], acc0, 0, 0, 0);
      acc1 = __builtin_amdgcn_mfma_f32_16x16x4f32(ac[k][1], b[1], acc1, 0, 0, 0);
      acc0 = __builtin_amdgcn_mfma_f32_16x16x4f32(ac[k][2], b[2], acc0, 0, 0, 0);
      acc1 = __builtin_amdgcn_mfma_f32_16x16x4f32(ac[k][3], b[3], acc1, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = acc0[i] + acc1[i];
  }
  if (fin)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (row + i < dk && col < dv) fin[io + (int64_t)i * dv] = s[i];
}

// O of a chunk for 64 columns of v.
template <typename T>
__global__ void __launch_bounds__(kThreads) delta_output_kernel(const DeltaParams p) {
  __shared__ __attribute__((aligned(16))) float qs[kTile], ks[kTile], ss[kTile];
  __shared__ __attribute__((aligned(16))) Gates gt;
  const int nvb = (p.dvp + 63) / 64, vb = 64 * (int)(blockIdx.x % nvb);
  const int64_t chunk = blockIdx.x / nvb;
  const At w = chunk_at(p, chunk);
  const int r0 = 16 * (threadIdx.x >> 6), hk = w.h / (p.H / p.Hk), vw = min(64, p.dvp - vb);
  T* const o = row_ptr<T>(p.o, w.b, w.t0, w.h) + vb;
  const int rows = (int)min((int64_t)kDeltaChunk, p.S - w.t0);   // of the output
  if (w.rows == 0) {
    for (int e = threadIdx.x; e < 64 * 64; e += kThreads)
      if ((e >> 6) < rows && vb + (e & 63) < p.dv_) o[(e >> 6) * p.o.ss + (e & 63)] = (T)0.0f;
    return;
  }
  load_gates(&gt, p.g, p.beta, w.b, w.t0, w.h, w.rows);
  const T* const q = row_ptr<T>(p.q, w.b, w.t0, hk);
  const T* const k = row_ptr<T>(p.k, w.b, w.t0, hk);
  const T* const v = row_ptr<T>(p.v, w.b, w.t0, w.h) + vb;
  const bool vec = p.vec;
  f32x4 P[4], kS[4], qS[4], x[4], acc[4];
  clear(P);
  clear(kS);
  clear(qS);
  for (int kb = 0; kb < p.dkp; kb += 64) {
    const int kw = min(64, p.dkp - kb);
    if (kb) __syncthreads();
    load_tile<kThreads>(ks, k + kb, p.k.ss, w.rows, p.dk_ - kb, kw, vec);
    load_tile<kThreads>(qs, q + kb, p.q.ss, w.rows, p.dk_ - kb, kw, vec);
    load_ws<kThreads>(ss, p.s + chunk * p.dkp * p.dvp + (int64_t)kb * p.dvp + vb, p.dvp, kw, vw);
    __syncthreads();
    mma<4, false, true>(P, qs, r0, ks, 0, 0, kw);
    mma<4, false, false>(kS, ks, r0, ss, 0, 0, kw);
    mma<4, false, false>(qS, qs, r0, ss, 0, 0, kw);
  }
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = out_row(r0, i), col = out_col(0, c);
      const bool in = row < w.rows && col < vw && vb + col < p.dv_;
      // (columns past vw hold what the tile had before: they are not stored)
      x[c][i] = in ? (float)v[row * p.v.ss + col] - gt.gam[row] * kS[c][i] : 0.0f;
      P[c][i] = row >= col ? P[c][i] * decay_between(gt, row, col) : 0.0f;
    }
  __syncthreads();
  put(qs, P, r0, 0);
  put(ss, x, r0, 0);
  load_ws<kThreads>(ks, p.z + chunk * 4096, 64, 64, 64);
  __syncthreads();
  clear(acc);
  mma<4, false, false, true>(acc, ks, r0, ss, 0, 0, r0 + 16, gt.beta);
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) x[c][i] = gt.beta[out_row(r0, i)] * (x[c][i] - acc[c][i]);
  __syncthreads();
  put(ss, x, r0, 0);
  __syncthreads();
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[c][i] = gt.gam[out_row(r0, i)] * qS[c][i];
  mma<4, false, false>(acc, qs, r0, ss, 0, 0, r0 + 16);
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = out_row(r0, i), col = out_col(0, c);
      if (row < rows && col < vw && vb + col < p.dv_)
        o[row * p.o.ss + col] = (T)(row < w.rows ? p.scale * acc[c][i] : 0.0f);
    }
}

template <typename T>
hipError_t forward(const DeltaParams& p, hipStream_t stream) {
  const int64_t chunks = (int64_t)p.B * p.H * p.N;
  hipLaunchKernelGGL((delta_prepare_kernel<T>), dim3((unsigned)chunks), dim3(kThreads), 0, stream, p);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess) e = launch_delta_scan(p, p.a, p.s, p.init, p.fin, false, stream);
  if (e != hipSuccess) return e;
  const int nvb = (p.dvp + 63) / 64;
  hipLaunchKernelGGL((delta_output_kernel<T>), dim3((unsigned)(chunks * nvb)), dim3(kThreads), 0, stream, p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_delta_scan(const DeltaParams& p, const float* a, float* x, const float* init, float* fin,
                             bool reverse, hipStream_t stream) {
  const int BH = p.B * p.H, ns = p.dvp / kDeltaSlice;
  const dim3 grid((unsigned)(8 * (int64_t)ns * ((BH + 7) / 8)));
  auto go = [&](auto kt) {
    constexpr int KT = decltype(kt)::value;
    hipLaunchKernelGGL((delta_scan_kernel<KT>), grid, dim3(64 * KT), 0, stream, a, x, init, fin, p.lengths, p.S, p.N,
                       BH, p.H, p.dk_, p.dv_, p.dvp, reverse);
  };
  switch (p.dkp / 16) {
    case 1: go(std::integral_constant<int, 1>{}); break;
    case 2: go(std::integral_constant<int, 2>{}); break;
    case 3: go(std::integral_constant<int, 3>{}); break;
    case 4: go(std::integral_constant<int, 4>{}); break;
    case 5: go(std::integral_constant<int, 5>{}); break;
    case 6: go(std::integral_constant<int, 6>{}); break;
    case 7: go(std::integral_constant<int, 7>{}); break;
    default: go(std::integral_constant<int, 8>{}); break;
  }
  return hipGetLastError();
}

hipError_t launch_delta_fwd(const DeltaParams& p, int dtype, hipStream_t stream) {
  return dtype == 0 ? forward<float>(p, stream) : forward<__bf16>(p, stream);
}

}  // namespace osm
