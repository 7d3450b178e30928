// The gated delta rule on gfx950: backward of the chunked forward (osm_delta.hip).
//
// Given a chunk's Z and start state S (saved by the forward), dO and D = dL/dS'
// of its end state (the names of osm_delta.hip; U = beta Y):
//   dU = scale P^T dO + Kt D,  R = dU - Z^T (beta dU),  dY = dV = beta R,  dbeta = R . Y
//   dP = scale dO U^T,  dL = -dY U^T          (on their triangles)
//   dQ  = scale e^G dO S^T + (dP o M) K
//   dKr = (dL o M) K - e^G dY S^T             k where it reads the state
//   dKw = (dP o M)^T Q + (dL o M)^T K + e^{G_last - G} U D^T   where it is written
//   dL/dS = A^T D + E,  E = (scale e^G Q - scale P W)^T dO
// g_t decays what tokens i >= t and the end state see of the start state and of
// tokens j < t, so, with the first terms of dQ and dKr and the last of dKw,
//   dg_t = sum_{i>=t} (q.dQ + k.dKr)_i + sum_{i>=t, j<t} C_ij + sum_{j<t} (k.dKw)_j + e^{G_last} <D, S>
//   C = dP o M o Q K^T + dL o M o K K^T
// (the sum from the right of dL/dG, with what cancels in it left out: pairs on
// one side of t never enter).
//
// Three launches: `adjoint` forms A^T and E of every chunk at once, the scan of
// the forward walks the chunks in reverse (every chunk's D over its E), and
// `grads` forms the gradients of every chunk at once.  q/k heads that several
// heads share get a gradient a head in fp32, which `fold` adds in order.
#include "osm_delta.h"

namespace osm {
namespace {

using namespace delta;

constexpr int kThreads = 256;

// Q K^T and, with KK, K K^T of a chunk on this wave's 16 rows; leaves the last
// blocks of q and k in qs and ks.
template <int NT, bool KK, int CT, typename T>
__device__ __forceinline__ void scores(f32x4 (&qk)[CT], f32x4 (&kk)[CT], float* qs, float* ks, const T* q, const T* k,
                                       const DeltaParams& p, int rows, int r0, int c0) {
  clear(qk);
  clear(kk);
  for (int kb = 0; kb < p.dkp; kb += 64) {
    const int kw = min(64, p.dkp - kb);
    if (kb) __syncthreads();
    load_tile<NT>(ks, k + kb, p.k.ss, rows, p.dk_ - kb, kw, p.vec == 4);
    load_tile<NT>(qs, q + kb, p.q.ss, rows, p.dk_ - kb, kw, p.vec == 4);
    __syncthreads();
    mma<CT, false, true>(qk, qs, r0, ks, c0, 0, kw);
    if (KK) mma<CT, false, true>(kk, ks, r0, ks, c0, 0, kw);
  }
}

// A^T and E of a chunk.
template <typename T>
__global__ void __launch_bounds__(kThreads) delta_adjoint_kernel(const DeltaParams p) {
  __shared__ __attribute__((aligned(16))) float zs[kTile], ps[kTile], ks[kTile], ws[kTile];
  __shared__ __attribute__((aligned(16))) Gates gt;
  const int64_t chunk = blockIdx.x;
  const At w = chunk_at(p, chunk);
  if (w.rows == 0) return;
  const int r0 = 16 * (threadIdx.x >> 6), hk = w.h / (p.H / p.Hk);
  load_gates(&gt, p.g, p.beta, w.b, w.t0, w.h, w.rows);
  const T* const q = row_ptr<T>(p.q, w.b, w.t0, hk);
  const T* const k = row_ptr<T>(p.k, w.b, w.t0, hk);
  const T* const go = row_ptr<T>(p.dout, w.b, w.t0, w.h);
  load_z<kThreads>(zs, p.z + chunk * kZFloats);
  f32x4 P[4], acc[4], x[4];
  scores<kThreads, false>(P, acc, ws, ks, q, k, p, w.rows, r0, 0);
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = out_row(r0, i), col = out_col(0, c);
      P[c][i] = row >= col ? P[c][i] * decay_between(gt, row, col) : 0.0f;
    }
  put(ps, P, r0, 0);
  const int nkb = (p.dkp + 63) / 64;
  float* const ag = p.a + chunk * p.dkp * p.dkp;
  float* const eg = p.d + chunk * p.dkp * p.dvp;
  for (int cb = 0; cb < nkb; ++cb) {
    const int cw = min(64, p.dkp - 64 * cb);
    __syncthreads();
    if (nkb > 1) load_tile<kThreads>(ks, k + 64 * cb, p.k.ss, w.rows, p.dk_ - 64 * cb, cw, p.vec == 4);
    __syncthreads();
    // W and, scaled to the chunk's end, its product with K: columns cb of Kt^T W,
    // so rows cb of A^T.
    clear(acc);
    mma<4, false, false, true>(acc, zs, r0, ks, 0, 0, r0 + 16, gt.bgam);
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = out_row(r0, i), col = out_col(0, c);
        x[c][i] = col < cw ? gt.beta[row] * (gt.gam[row] * ks[row * kLd + col] - acc[c][i]) : 0.0f;
        acc[c][i] = gt.end[row] * x[c][i];
      }
    put(ws, acc, r0, 0);
    __syncthreads();
    for (int rb = 0; rb < nkb; ++rb) {
      const int rw = min(64, p.dkp - 64 * rb);
      if (nkb > 1) {
        __syncthreads();
        load_tile<kThreads>(ks, k + 64 * rb, p.k.ss, w.rows, p.dk_ - 64 * rb, rw, p.vec == 4);
        __syncthreads();
      }
      if (r0 < cw) {
        clear(acc);
        mma<4, true, false>(acc, ws, r0, ks, 0, 0, 64);
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = 64 * cb + out_row(r0, i), col = out_col(0, c);
            if (col < rw)
              ag[(int64_t)row * p.dkp + 64 * rb + col] = (row == 64 * rb + col ? gt.last : 0.0f) - acc[c][i];
          }
      }
    }
    __syncthreads();
    // e^G Q - P W, by columns cb, and rows cb of E
    put(ws, x, r0, 0);
    __syncthreads();
    clear(acc);
    mma<4, false, false>(acc, ps, r0, ws, 0, 0, r0 + 16);
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = out_row(r0, i), col = out_col(0, c);
        const float qv = row < w.rows && 64 * cb + col < p.dk_ ? (float)q[row * p.q.ss + 64 * cb + col] : 0.0f;
        acc[c][i] = p.scale * (gt.gam[row] * qv - acc[c][i]);
      }
    __syncthreads();
    put(ws, acc, r0, 0);
    for (int vb = 0; vb < p.dvp; vb += 64) {
      const int vw = min(64, p.dvp - vb);
      __syncthreads();
      load_tile<kThreads>(ks, go + vb, p.dout.ss, w.rows, p.dv_ - vb, vw, p.vec == 4);
      __syncthreads();
      if (r0 < cw) {
        clear(acc);
        mma<4, true, false>(acc, ws, r0, ks, 0, 0, 64);
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int col = out_col(0, c);
            if (col < vw) eg[(int64_t)(64 * cb + out_row(r0, i)) * p.dvp + vb + col] = acc[c][i];
          }
      }
    }
  }
}

constexpr int kGradThreads = 512;

// The gradients of a chunk: eight waves, 16 rows by 32 columns of every product
// each; nine tiles of LDS (157 KB), one workgroup a CU.  NKB: blocks of 64
// columns of q and k.
template <typename T, int NKB>
__global__ void __launch_bounds__(kGradThreads) delta_grads_kernel(const DeltaParams p) {
  constexpr int CT = 2;
  __shared__ __attribute__((aligned(16))) float zs[kTile], ps[kTile], ks[kTile], qs[kTile], ss[kTile], ds[kTile],
      us[kTile], os[kTile], ys[kTile];
  __shared__ __attribute__((aligned(16))) Gates gt;
  // By column half: the reads' and the writes' parts of dg, dbeta; by wave: the
  // pairs' part of dg, <D, S>.
  __shared__ float row_sum[3][2][64], pairs[8][64], part[8];
  const int64_t chunk = blockIdx.x;
  const At w = chunk_at(p, chunk);
  const int tid = threadIdx.x, wave = tid >> 6, r0 = 16 * (wave & 3), c0 = 32 * (wave >> 2);
  const int hk = w.h / (p.H / p.Hk);
  const bool shared_heads = p.H != p.Hk;   // dq and dk are then fp32, by head
  const int rows = (int)min((int64_t)kDeltaChunk, p.S - w.t0);
  T* const gv = row_ptr<T>(p.dv, w.b, w.t0, w.h);
  auto put_qk = [&](const DeltaRows& dst, int row, int col, float v) {
    if (shared_heads)
      row_ptr<float>(dst, w.b, w.t0 + row, w.h)[col] = v;
    else
      row_ptr<T>(dst, w.b, w.t0 + row, w.h)[col] = (T)v;
  };
  auto put_gate = [&](const DeltaRows& dst, int row, float v) { *row_ptr<float>(dst, w.b, w.t0 + row, w.h) = v; };
  if (w.rows == 0) {
    for (int row = wave; row < rows; row += 8) {
      for (int e = tid & 63; e < p.dk_; e += 64) {
        put_qk(p.dq, row, e, 0.0f);
        put_qk(p.dk, row, e, 0.0f);
      }
      for (int e = tid & 63; e < p.dv_; e += 64) gv[row * p.dv.ss + e] = (T)0.0f;
      if ((tid & 63) == 0) {
        put_gate(p.dg, row, 0.0f);
        put_gate(p.dbeta, row, 0.0f);
      }
    }
    return;
  }
  load_gates(&gt, p.g, p.beta, w.b, w.t0, w.h, w.rows);
  load_z<kGradThreads>(zs, p.z + chunk * kZFloats);
  const T* const q = row_ptr<T>(p.q, w.b, w.t0, hk);
  const T* const k = row_ptr<T>(p.k, w.b, w.t0, hk);
  const T* const v = row_ptr<T>(p.v, w.b, w.t0, w.h);
  const T* const go = row_ptr<T>(p.dout, w.b, w.t0, w.h);
  const float* const sg = p.s + chunk * p.dkp * p.dvp;
  const float* const dg = p.d + chunk * p.dkp * p.dvp;
  f32x4 M[CT], qk[CT], kk[CT], dP[CT], dL[CT], x[CT], y[CT], acc[CT];
  f32x4 dq[NKB][CT], dkr[NKB][CT], dkw[NKB][CT];
  f32x4 reads = zero4(), writes = zero4(), bsum = zero4();   // of this wave's rows, its columns' part
  float ending = 0.0f;                                       // this thread's part of <D, S>
  scores<kGradThreads, true>(qk, kk, qs, ks, q, k, p, w.rows, r0, c0);
#pragma unroll
  for (int c = 0; c < CT; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = out_row(r0, i), col = out_col(c0, c);
      M[c][i] = row >= col ? decay_between(gt, row, col) : 0.0f;
      acc[c][i] = row >= col ? qk[c][i] * M[c][i] : 0.0f;
    }
  put(ps, acc, r0, c0);
  clear(dP);
  clear(dL);
#pragma unroll
  for (int b = 0; b < NKB; ++b) {
    clear(dq[b]);
    clear(dkr[b]);
    clear(dkw[b]);
  }
  auto width = [&](int b) { return min(64, p.dkp - 64 * b); };
  for (int vb = 0; vb < p.dvp; vb += 64) {
    const int vw = min(64, p.dvp - vb);
    __syncthreads();
    load_tile<kGradThreads>(os, go + vb, p.dout.ss, w.rows, p.dv_ - vb, 64, p.vec == 4);
    clear(x);
    clear(y);
#pragma unroll
    for (int b = 0; b < NKB; ++b) {
      if (b) __syncthreads();
      if (NKB > 1) load_tile<kGradThreads>(ks, k + 64 * b, p.k.ss, w.rows, p.dk_ - 64 * b, width(b), p.vec == 4);
      load_ws<kGradThreads>(ss, sg + (int64_t)64 * b * p.dvp + vb, p.dvp, width(b), vw);
      load_ws<kGradThreads>(ds, dg + (int64_t)64 * b * p.dvp + vb, p.dvp, width(b), vw);
      __syncthreads();
      mma<CT, false, false>(x, ks, r0, ss, c0, 0, width(b));
      mma<CT, false, false>(y, ks, r0, ds, c0, 0, width(b));
      float dot = 0.0f;
      for (int e = tid; e < width(b) * (vw >> 2); e += kGradThreads) {
        const int row = e / (vw >> 2), col = 4 * (e - row * (vw >> 2));
        const f32x4 a = load4(ss + row * kLd + col), d = load4(ds + row * kLd + col);
#pragma unroll
        for (int i = 0; i < 4; ++i) dot = __builtin_fmaf(a[i], d[i], dot);
      }
      ending += dot;
    }
    // X (zeros past the columns in use), and dU
    clear(acc);
    mma<CT, true, false>(acc, ps, r0, os, c0, r0, 64);
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = out_row(r0, i), col = out_col(c0, c);
        const bool in = row < w.rows && vb + col < p.dv_ && col < vw;
        x[c][i] = in ? (float)v[row * p.v.ss + vb + col] - gt.gam[row] * x[c][i] : 0.0f;
        y[c][i] = in ? p.scale * acc[c][i] + gt.end[row] * y[c][i] : 0.0f;
      }
    put(us, x, r0, c0);
    put(ys, y, r0, c0);
    __syncthreads();
    clear(acc);
    mma<CT, false, false, true>(acc, zs, r0, us, c0, 0, r0 + 16, gt.beta);
#pragma unroll
    for (int c = 0; c < CT; ++c) x[c] -= acc[c];           // Y
    clear(acc);
    mma<CT, true, false, true>(acc, zs, r0, ys, c0, r0, 64, gt.beta);
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = out_row(r0, i), col = out_col(c0, c);
        const float r = y[c][i] - acc[c][i], beta = gt.beta[row];
        bsum[i] = __builtin_fmaf(r, x[c][i], bsum[i]);
        x[c][i] *= beta;                                    // U
        y[c][i] = beta * r;                                 // dY
        if (row < rows && col < vw && vb + col < p.dv_) gv[row * p.dv.ss + vb + col] = (T)y[c][i];
      }
    __syncthreads();
    put(us, x, r0, c0);
    put(ys, y, r0, c0);
    __syncthreads();
    mma<CT, false, true>(dP, os, r0, us, c0, 0, vw);
    mma<CT, false, true>(dL, ys, r0, us, c0, 0, vw);
#pragma unroll
    for (int b = 0; b < NKB; ++b) {
      if (NKB > 1) {
        __syncthreads();
        load_tile<kGradThreads>(ks, k + 64 * b, p.k.ss, w.rows, p.dk_ - 64 * b, width(b), p.vec == 4);
        load_ws<kGradThreads>(ss, sg + (int64_t)64 * b * p.dvp + vb, p.dvp, width(b), vw);
        load_ws<kGradThreads>(ds, dg + (int64_t)64 * b * p.dvp + vb, p.dvp, width(b), vw);
        __syncthreads();
      }
      mma<CT, false, true>(dq[b], os, r0, ss, c0, 0, vw);
      mma<CT, false, true>(dkr[b], ys, r0, ss, c0, 0, vw);
      clear(acc);
      mma<CT, false, true>(acc, us, r0, ds, c0, 0, vw);
#pragma unroll
      for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = out_row(r0, i), col = out_col(c0, c);
          const float e = gt.end[row] * acc[c][i];
          if (col < width(b)) {
            dkw[b][c][i] += e;
            writes[i] = __builtin_fmaf(e, ks[row * kLd + col], writes[i]);
          }
        }
    }
  }
  // (dP o M) and (dL o M) take the places of P and Z, C that of dO
  __syncthreads();
#pragma unroll
  for (int c = 0; c < CT; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = out_row(r0, i), col = out_col(c0, c);
      dP[c][i] = row >= col ? p.scale * dP[c][i] * M[c][i] : 0.0f;
      dL[c][i] = row > col ? -dL[c][i] * M[c][i] : 0.0f;
      acc[c][i] = row > col ? dP[c][i] * qk[c][i] + dL[c][i] * kk[c][i] : 0.0f;
    }
  put(ps, dP, r0, c0);
  put(zs, dL, r0, c0);
  put(os, acc, r0, c0);
  __syncthreads();
  {
    // Wave w sums C over its rows i in [8w, 8w + 8) for every t, lane t: over
    // j < t by a scan along the row, then over the rows at and past t.
    const int t = tid & 63;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int row = 8 * wave + i;
      float v = os[row * kLd + t];
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const float up = __shfl_up(v, o);
        if (t >= o) v += up;
      }
      const float before = __shfl_up(v, 1);   // sum_{j < t}
      if (t > 0 && row >= t) sum += before;
    }
    pairs[wave][t] = sum;
  }
#pragma unroll
  for (int b = 0; b < NKB; ++b) {
    if (NKB > 1) {
      if (b) __syncthreads();
      load_tile<kGradThreads>(ks, k + 64 * b, p.k.ss, w.rows, p.dk_ - 64 * b, width(b), p.vec == 4);
      load_tile<kGradThreads>(qs, q + 64 * b, p.q.ss, w.rows, p.dk_ - 64 * b, width(b), p.vec == 4);
      __syncthreads();
    }
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float gam = gt.gam[out_row(r0, i)];
        dq[b][c][i] *= p.scale * gam;
        dkr[b][c][i] *= -gam;
      }
    if (c0 >= width(b)) continue;   // (the barriers above are behind every wave)
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = out_row(r0, i) * kLd + out_col(c0, c);
        if (out_col(c0, c) < width(b)) reads[i] += qs[at] * dq[b][c][i] + ks[at] * dkr[b][c][i];
      }
    mma<CT, false, false>(dq[b], ps, r0, ks, c0, 0, r0 + 16);
    mma<CT, false, false>(dkr[b], zs, r0, ks, c0, 0, r0 + 16);
    mma<CT, true, false>(dkw[b], ps, r0, qs, c0, r0, 64);
    mma<CT, true, false>(dkw[b], zs, r0, ks, c0, r0, 64);
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = out_row(r0, i), col = out_col(c0, c);
        if (col < width(b) && 64 * b + col < p.dk_) {
          if (row < rows) {
            put_qk(p.dq, row, 64 * b + col, dq[b][c][i]);
            put_qk(p.dk, row, 64 * b + col, dkr[b][c][i] + dkw[b][c][i]);
          }
        }
      }
  }
  // The rows' sums: the sixteen columns of a tile by shuffle, the halves in order.
#pragma unroll
  for (int o = 1; o < 16; o <<= 1)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      reads[i] += __shfl_xor(reads[i], o);
      writes[i] += __shfl_xor(writes[i], o);
      bsum[i] += __shfl_xor(bsum[i], o);
    }
  if ((tid & 15) == 0)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      row_sum[0][wave >> 2][out_row(r0, i)] = reads[i];
      row_sum[1][wave >> 2][out_row(r0, i)] = writes[i];
      row_sum[2][wave >> 2][out_row(r0, i)] = bsum[i];
    }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) ending += __shfl_xor(ending, o);
  if ((tid & 63) == 0) part[wave] = ending;
  __syncthreads();
  if (tid < 64) {
    float from = row_sum[0][0][tid] + row_sum[0][1][tid], upto = row_sum[1][0][tid] + row_sum[1][1][tid];
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const float down = __shfl_down(from, o), up = __shfl_up(upto, o);
      if (tid + o < 64) from += down;
      if (tid >= o) upto += up;
    }
    upto = __shfl_up(upto, 1);
    float sum = from + (tid > 0 ? upto : 0.0f), whole = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      sum += pairs[i][tid];
      whole += part[i];
    }
    if (tid < rows) {
      put_gate(p.dg, tid, tid < w.rows ? sum + gt.last * whole : 0.0f);
      put_gate(p.dbeta, tid, tid < w.rows ? row_sum[2][0][tid] + row_sum[2][1][tid] : 0.0f);
    }
  }
}

// dst[b,t,hk,:] = the sum over the heads that share hk, in order, of src [B,S,H,dk].
template <typename T>
__global__ void __launch_bounds__(kThreads) delta_fold_kernel(const float* src, DeltaRows dst, int64_t n, int S, int Hk,
                                                              int group, int dk) {
  const int64_t e = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (e >= n) return;
  const int j = (int)(e % dk);
  const int64_t hb = e / dk;            // (b S + t) Hk + hk
  const float* p = src + hb * group * dk + j;
  float s = p[0];
  for (int i = 1; i < group; ++i) s += p[(int64_t)i * dk];
  const int64_t bt = hb / Hk;
  row_ptr<T>(dst, bt / S, bt % S, hb % Hk)[j] = (T)s;
}

template <typename T>
hipError_t backward(const DeltaParams& p, float* const part, hipStream_t stream) {
  const unsigned chunks = (unsigned)((int64_t)p.B * p.H * p.N);
  hipLaunchKernelGGL((delta_adjoint_kernel<T>), dim3(chunks), dim3(kThreads), 0, stream, p);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess) e = launch_delta_scan(p, p.a, p.d, p.grad_state, p.grad_init, p.N, kDeltaChunk, true, stream);
  if (e != hipSuccess) return e;
  const int64_t plane = (int64_t)p.B * p.S * p.H * p.dk_;
  DeltaParams w = p;
  if (p.H != p.Hk) {
    const DeltaRows own = {nullptr, (int64_t)p.S * p.H * p.dk_, (int64_t)p.H * p.dk_, p.dk_};
    w.dq = w.dk = own;
    w.dq.p = part;
    w.dk.p = part + plane;
  }
  if (p.dkp <= 64)
    hipLaunchKernelGGL((delta_grads_kernel<T, 1>), dim3(chunks), dim3(kGradThreads), 0, stream, w);
  else
    hipLaunchKernelGGL((delta_grads_kernel<T, 2>), dim3(chunks), dim3(kGradThreads), 0, stream, w);
  e = hipGetLastError();
  if (e != hipSuccess || p.H == p.Hk) return e;
  const int64_t n = (int64_t)p.B * p.S * p.Hk * p.dk_;
  const dim3 grid((unsigned)((n + kThreads - 1) / kThreads));
  hipLaunchKernelGGL((delta_fold_kernel<T>), grid, dim3(kThreads), 0, stream, part, p.dq, n, p.S, p.Hk, p.H / p.Hk,
                     p.dk_);
  hipLaunchKernelGGL((delta_fold_kernel<T>), grid, dim3(kThreads), 0, stream, part + plane, p.dk, n, p.S, p.Hk,
                     p.H / p.Hk, p.dk_);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_delta_bwd(const DeltaParams& p, float* part, int dtype, hipStream_t stream) {
  return dtype == 0 ? backward<float>(p, part, stream) : backward<__bf16>(p, part, stream);
}

}  // namespace osm
