// The gated delta rule on gfx950: backward of the chunked forward (osm_delta.hip).
//
// Given a chunk's Z and start state S (saved by the forward), dO and D = dL/dS'
// of its end state (the names of osm_delta.hip; U = beta Y):
//   dU = scale P^T dO + Kt D,  R = dU - Z^T (beta dU),  dY = dV = beta R,  dbeta = R . Y
//   dP = scale dO U^T,  dL = -dY U^T          (on their triangles)
//   dQ  = scale e^G dO S^T + (dP o M) K
//   dKr = (dL o M) K - e^G dY S^T             k where it reads the state
//   dKw = (dP o M)^T Q + (dL o M)^T K + e^{G_last - G} U D^T   where it is written
//   dL/dS = e^{G_last} D + Q^T (scale e^G dO) - K^T (e^G dY)
// g_t decays what tokens i >= t and the end state see of the start state and of
// tokens j < t, so, with the first terms of dQ and dKr and the last of dKw,
//   dg_t = sum_{i>=t} (q.dQ + k.dKr)_i + sum_{i>=t, j<t} C_ij + sum_{j<t} (k.dKw)_j + e^{G_last} <D, S>
//   C = dP o M o Q K^T + dL o M o K K^T
// (the sum from the right of dL/dG, with what cancels in it left out: pairs on
// one side of t never enter).
//
// Launches: `rewalk` walks the segments of the forward's walk in reverse with D in
// the waves' accumulators, giving dV and leaving every chunk's D (where a row has
// several segments, a first walk gives their maps of D and the scan joins them),
// and `grads` forms the other gradients of every chunk at once.  q/k heads that
// several heads share get a gradient a head in fp32, which `fold` adds in order.
#include <type_traits>

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

// As tri_at's matrices, for the transpose: rows 0-31 have 64 columns, the others
// the last 32.
__device__ __forceinline__ int upper_at(int row, int col) { return row < 32 ? row * 72 + col : 2304 + (row - 32) * 40 + col - 32; }

// Walks segment blockIdx.x % segs of a head from its last chunk to its first, D =
// dL/dS' in the waves' accumulators (16 columns each, as S in the forward's walk).
// MAP: the segment's map of D; else dV, and every chunk's D into p.d.  What bounds
// it is what bounds the forward's walk (64 chunks of 32 heads, bf16, d = 64: 59 us
// for the maps, 43 for dV).  Four waves instead of eight for the maps lost 10 to 60
// us of a backward there, and won 13 only where dk = 32, dv = 128.
template <typename T, int KS, int WAVES, bool MAP>
__global__ void __launch_bounds__(64 * WAVES, 2) delta_rewalk_kernel(const DeltaParams p, int groups) {
  constexpr int NT = 64 * WAVES, NP = kParts<T>, DK = 32 * KS, LDK = DK + 8, LKT = 72, ST = 2 * KS;
  // K and Q by rows, then both by columns in the same place.
  constexpr int kK = 64 * LDK, kKt = DK * LKT, kOne = kK > kKt ? kK : kKt;
  __shared__ __attribute__((aligned(16))) unsigned short in[NP][2 * kOne], zt[3][kTri], pt[3][kTri];
  __shared__ __attribute__((aligned(16))) float gates[2][kGateFloats];
  unsigned short *const kk = &in[0][0], *const qq = kk + kOne;
  constexpr int kIn = 2 * kOne;
  const int group = blockIdx.x % groups;
  const int64_t id = blockIdx.x / groups;
  const int seg = (int)(id % p.segs), bh = (int)(id / p.segs), b = bh / p.H, h = bh - b * p.H, hk = h / (p.H / p.Hk);
  const int tid = threadIdx.x, wave = tid >> 6, l = tid & 63, r = l & 15, g = l >> 4;
  const int tokens = p.lengths ? min(max(p.lengths[b], 0), p.S) : p.S;
  const int n = (tokens + kDeltaChunk - 1) / kDeltaChunk;
  const int c0 = seg * p.seg, c1 = min(min(c0 + p.seg, p.N), n);
  const int slice = group * WAVES + wave, vs = p.dvp / kDeltaSlice;
  const bool value = slice < vs, live = slice < vs + (MAP ? DK / kDeltaSlice : 0);
  const int col = kDeltaSlice * slice + r;
  const bool in_v = value && col < p.dv_;
  const bool first = !MAP && p.grad_init && seg == 0;
  if (!MAP) {
    // zeros for the chunks without tokens
    for (int c = max(c0, n); c < min(c0 + p.seg, p.N); ++c) {
      T* const o = row_ptr<T>(p.dv, b, (int64_t)c * kDeltaChunk, h) + col;
      if (in_v)
        for (int t = g; t < min(kDeltaChunk, p.S - c * kDeltaChunk); t += 4) o[t * p.dv.ss] = (T)0.0f;
    }
  }
  if (c0 >= c1 && !first) return;
  if (MAP && c0 == 0) return;   // nothing comes before the first segment
  f32x4 D[ST];
  const bool ws = !MAP && p.segs > 1 && n > 0;
  const float* const from =
      MAP ? nullptr : ws ? p.x + id * DK * p.dvp : p.grad_state ? p.grad_state + (int64_t)bh * p.dk_ * p.dv_ : nullptr;
  const Rsrc from_rs = make_rsrc(from);
  const unsigned from_ld = 4u * (ws ? p.dvp : p.dv_);
  const bool from_col = from && (ws ? value : in_v);
#pragma unroll
  for (int t = 0; t < ST; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 16 * t + 4 * g + i;
      if (MAP)
        D[t][i] = !value && row == col - p.dvp ? 1.0f : 0.0f;
      else
        D[t][i] = raw_value<float>(load_raw<float>(from_rs, from_col && (ws || row < p.dk_) ? row * from_ld + 4u * col : kOut));
    }
  const T* const kp = row_ptr<T>(p.k, b, 0, hk);
  const T* const qp = row_ptr<T>(p.q, b, 0, hk);
  const T* const dop = row_ptr<T>(p.dout, b, 0, h);
  T* const dvp = MAP ? nullptr : row_ptr<T>(p.dv, b, 0, h);
  const unsigned es = sizeof(T), do_row = (unsigned)p.dout.ss * es, dv_row = (unsigned)p.dv.ss * es;
  const unsigned do_at = in_v ? col * es + 4 * g * do_row : kOut, dv_at = in_v ? col * es + 4 * g * dv_row : kOut;
  // Z by 4x4 blocks: 64 of rows 0-31, then 128
  const int zi = tid < 64 ? 4 * (tid >> 3) : 32 + 4 * ((tid - 64) >> 4), zj = 4 * (tid < 64 ? tid & 7 : (tid - 64) & 15);
  Block<T, KS, NT> kb, qb;
  f32x4 zr[4];
  unsigned dr[16];
  float gr[2];
  auto rows_of = [&](int c) { return min(kDeltaChunk, tokens - c * kDeltaChunk); };
  auto fetch_kq = [&](int c) {
    kb.load(kp + (int64_t)c * kDeltaChunk * p.k.ss, p.k.ss, rows_of(c), p.dk_, p.vec);
    qb.load(qp + (int64_t)c * kDeltaChunk * p.q.ss, p.q.ss, rows_of(c), p.dk_, p.vec);
  };
  auto fetch_do = [&](int c) {
    const Rsrc rs = rows_rsrc<T>(dop + (int64_t)c * kDeltaChunk * p.dout.ss, p.dout.ss, rows_of(c), p.dv_);
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) dr[4 * t + i] = load_raw<T>(rs, do_at, (16 * t + i) * do_row);
  };
  auto fetch = [&](int c) {
    const int64_t chunk = (int64_t)bh * p.N + c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = min(zi, 60) + i, quad = row < 32 ? row * 8 + (zj >> 2) : 256 + (row - 32) * 16 + (zj >> 2);
      zr[i] = load4(p.z + chunk * kZFloats + 4 * quad);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) gr[e] = p.gates[chunk * kGateFloats + min(tid + e * NT, kGateFloats - 1)];
  };
  auto put_gates = [&](int c) {
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (tid + e * NT < kGateFloats) gates[c & 1][tid + e * NT] = gr[e];
  };
  if (c0 < c1) {
    fetch_kq(c1 - 1);
    fetch(c1 - 1);
    fetch_do(c1 - 1);
    put_gates(c1 - 1);
    // P's zeros before the diagonal tiles that end a pair: rows 16-31 and 48-63
    for (int e = tid; e < 32 * 3 * 4; e += NT) {
      const int row = (e & 31) < 16 ? 16 + (e & 31) : 32 + (e & 31), k = (e >> 5) % 3, q = 4 * (row >> 5 << 1) + (e >> 5) / 3;
      *reinterpret_cast<u32x2*>(&pt[k][upper_at(row, place4(q))]) = u32x2{0, 0};
    }
  }
  for (int c = c1 - 1; c >= c0; --c) {
    const int64_t t0 = (int64_t)c * kDeltaChunk;
    const float* const gt = gates[c & 1];
    __syncthreads();   // the chunk after has been read, this one's gates are there
    kb.template put_rows<LDK>(kk, kIn);
    qb.template put_rows<LDK>(qq, kIn);
    if (tid < 192) {
      // -(beta Z)^T
#pragma unroll
      for (int i = 0; i < 4; ++i) zr[i] *= -gt[kBeta + zi + i];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        u32x2 part[3];
        split4<3>(part, f32x4{zr[0][j], zr[1][j], zr[2][j], zr[3][j]});
#pragma unroll
        for (int k = 0; k < 3; ++k) *reinterpret_cast<u32x2*>(&zt[k][upper_at(zj + j, place4(zi >> 2))]) = part[k];
      }
    }
    __syncthreads();
    if (c > c0) fetch(c - 1);
    // scale P^T: four of its columns (rows of Q) of one row a lane
#pragma unroll
    for (int e = 0; e < (9 + WAVES) / WAVES; ++e) {
      const int tile = wave + WAVES * e;
      if (tile < 10) {
        const int ti = tile < 1 ? 0 : tile < 3 ? 1 : tile < 6 ? 2 : 3, tj = tile - ti * (ti + 1) / 2, j = 16 * tj + r;
        f32x4 acc = zero4();
        u32x4 kf[KS][NP], qf[KS][NP];
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          read_parts<NP>(qf[s], qq, kIn, (16 * ti + r) * LDK + 32 * s + 8 * g);
          read_parts<NP>(kf[s], kk, kIn, j * LDK + 32 * s + 8 * g);
        }
#pragma unroll
        for (int s = 0; s < KS; ++s) mul<NP, 2>(acc, qf[s], kf[s]);
        const f32x4 hi = load4(gt + kHi + 16 * ti + 4 * g), lo = load4(gt + kLo + 16 * ti + 4 * g);
        const float hi_j = gt[kHi + j], lo_j = gt[kLo + j];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          acc[k] = 16 * ti + 4 * g + k >= j ? p.scale * acc[k] * __builtin_amdgcn_exp2f((hi[k] - hi_j) + (lo[k] - lo_j)) : 0.0f;
        u32x2 part[3];
        split4<3>(part, acc);
#pragma unroll
        for (int k = 0; k < 3; ++k) *reinterpret_cast<u32x2*>(&pt[k][upper_at(j, place4(4 * ti + g))]) = part[k];
      }
    }
    f32x4 x[4];
    u32x4 dp[2][NP];   // dO
    if (live) {
      if (!MAP && value) {
        float* const dg = p.d + ((int64_t)bh * p.N + c) * DK * p.dvp + col;
#pragma unroll
        for (int t = 0; t < ST; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) dg[(int64_t)(16 * t + 4 * g + i) * p.dvp] = D[t][i];
      }
      clear(x);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        u32x4 sp[3];
        split_pair<3>(sp, D[2 * s], D[2 * s + 1]);
        products<NP, (NP == 1 ? 3 : 1), 4>(
            kIn, [&](int i) { return kk + (16 * i + r) * LDK + 32 * s + 8 * g; },
            [&](int i, const u32x4(&a)[NP]) { mul<3, 2>(x[i], a, sp); });
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) x[t] *= load4(gt + kEnd + 16 * t + 4 * g);
    }
    __syncthreads();   // P is there, the rows have been read
    kb.template put_columns<LKT>(kk, kIn);
    qb.template put_columns<LKT>(qq, kIn);
    if (c > c0) fetch_kq(c - 1);
    if (live) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        if constexpr (NP == 1)
          dp[s][0] = u32x4{dr[8 * s] | dr[8 * s + 1] << 16, dr[8 * s + 2] | dr[8 * s + 3] << 16,
                           dr[8 * s + 4] | dr[8 * s + 5] << 16, dr[8 * s + 6] | dr[8 * s + 7] << 16};
        else
          split_pair<NP>(dp[s], f32x4{raw_value<T>(dr[8 * s]), raw_value<T>(dr[8 * s + 1]), raw_value<T>(dr[8 * s + 2]), raw_value<T>(dr[8 * s + 3])},
                         f32x4{raw_value<T>(dr[8 * s + 4]), raw_value<T>(dr[8 * s + 5]), raw_value<T>(dr[8 * s + 6]), raw_value<T>(dr[8 * s + 7])});
      }
      // tiles (t, s): (0, 0), (1, 0), (0, 1) .. (3, 1)
      products<3, 1, 6>(
          kTri, [&](int i) { return &pt[0][0] + upper_at(16 * (i < 2 ? i : i - 2) + r, 32 * (i >= 2) + 8 * g); },
          [&](int i, const u32x4(&a)[3]) { mul<NP, 2>(x[i < 2 ? i : i - 2], a, dp[i >= 2]); });
      // R, on R0's registers
      u32x4 xp[2][3];
      split_pair<3>(xp[0], x[0], x[1]);
      split_pair<3>(xp[1], x[2], x[3]);
      products<3, 1, 6>(
          kTri, [&](int i) { return &zt[0][0] + upper_at(16 * (i < 2 ? i : i - 2) + r, 32 * (i >= 2) + 8 * g); },
          [&](int i, const u32x4(&a)[3]) { mul<3, 2>(x[i < 2 ? i : i - 2], a, xp[i >= 2]); });
#pragma unroll
      for (int t = 0; t < 4; ++t) x[t] *= load4(gt + kBeta + 16 * t + 4 * g);   // dY
      if (!MAP) {
        const int rows = tokens - (int)t0;
        if (rows < kDeltaChunk)   // zeros past the tokens in use
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (16 * t + 4 * g + i >= rows) x[t][i] = 0.0f;
        const Rsrc o_rs = rows_rsrc<T>(dvp + t0 * p.dv.ss, p.dv.ss, min(kDeltaChunk, p.S - (int)t0), p.dv_);
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) store_one<T>(o_rs, dv_at, (16 * t + i) * dv_row, x[t][i]);
      }
    }
    __syncthreads();   // the columns are there
    if (live) {
      const float last = gt[kGam + 63];
#pragma unroll
      for (int t = 0; t < ST; ++t) D[t] *= last;
      f32x4 gam[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) gam[t] = load4(gt + kGam + 16 * t + 4 * g);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        u32x4 yp[3], op[3];
        split_pair<3>(yp, -x[2 * s] * gam[2 * s], -x[2 * s + 1] * gam[2 * s + 1]);
        f32x4 o[2];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[t][i] = p.scale * gam[2 * s + t][i] * raw_value<T>(dr[8 * s + 4 * t + i]);
        split_pair<3>(op, o[0], o[1]);
        products<NP, (NP == 1 ? 3 : 1), 2 * ST>(
            kIn, [&](int i) { return (i < ST ? kk : qq) + (16 * (i % ST) + r) * LKT + 32 * s + 8 * g; },
            [&](int i, const u32x4(&a)[NP]) { mul<3, 2>(D[i % ST], a, i < ST ? yp : op); });
      }
    }
    if (c > c0) {
      fetch_do(c - 1);
      put_gates(c - 1);
    }
  }
  if (MAP && live) {
    float* const dst = value ? p.x + id * DK * p.dvp + col : p.a + id * DK * DK + (col - p.dvp);
    const int ld = value ? p.dvp : DK;
#pragma unroll
    for (int t = 0; t < ST; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) dst[(int64_t)(16 * t + 4 * g + i) * ld] = D[t][i];
  }
  if (first && in_v) {
    float* const dst = p.grad_init + (int64_t)bh * p.dk_ * p.dv_ + col;
#pragma unroll
    for (int t = 0; t < ST; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (16 * t + 4 * g + i < p.dk_) dst[(int64_t)(16 * t + 4 * g + i) * p.dv_] = D[t][i];
  }
}

template <typename T, int KS, bool MAP>
void launch_rewalk(const DeltaParams& p, hipStream_t stream) {
  const int slices = p.dvp / kDeltaSlice + (MAP ? p.dkp / kDeltaSlice : 0);
  auto go = [&](auto waves) {
    constexpr int W = decltype(waves)::value;
    const int groups = (slices + W - 1) / W;
    const unsigned grid = (unsigned)((int64_t)p.B * p.H * p.segs * groups);
    hipLaunchKernelGGL((delta_rewalk_kernel<T, KS, W, MAP>), dim3(grid), dim3(64 * W), 0, stream, p, groups);
  };
  if (slices <= 4)
    go(std::integral_constant<int, 4>{});
  else
    go(std::integral_constant<int, 8>{});
}

constexpr int kGradThreads = 512;

// The gradients of a chunk but dV, from fp32 inputs, on the fp32 matrix
// instruction: eight waves, 16 rows by 32 columns of every product each; nine tiles
// of LDS (157 KB), one workgroup a CU.  NKB: blocks of 64 columns of q and k.  What
// bounds it: the matrix instructions and the barriers between the products (376
// chunks of dk = 48, dv = 80: 85 us).
template <int NKB>
__global__ void __launch_bounds__(kGradThreads) delta_grads_kernel(const DeltaParams p) {
  typedef float T;
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
  const int rows = (int)min((int64_t)kDeltaChunk, p.S - w.t0);
  auto put_qk = [&](const DeltaRows& dst, int row, int col, float v) {
    row_ptr<T>(dst, w.b, w.t0 + row, w.h)[col] = v;   // (also where heads are shared: fp32, by head)
  };
  auto put_gate = [&](const DeltaRows& dst, int row, float v) { *row_ptr<float>(dst, w.b, w.t0 + row, w.h) = v; };
  if (w.rows == 0) {
    for (int row = wave; row < rows; row += 8) {
      for (int e = tid & 63; e < p.dk_; e += 64) {
        put_qk(p.dq, row, e, 0.0f);
        put_qk(p.dk, row, e, 0.0f);
      }
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
        x[c][i] = in ? v[row * p.v.ss + vb + col] - gt.gam[row] * x[c][i] : 0.0f;
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

// ---- bf16 inputs ----

// Four elements of a row from `at` (kOut: zeros), `left` of them inside it.
__device__ __forceinline__ bf16x4 load_quad(Rsrc rs, unsigned at, int left, int vec) {
  if (vec == 4) return __builtin_bit_cast(bf16x4, __builtin_amdgcn_raw_buffer_load_b64(rs, left > 0 ? at : kOut, 0, 0));
  if (vec == 2)
    return __builtin_bit_cast(bf16x4, u32x2{__builtin_amdgcn_raw_buffer_load_b32(rs, left > 0 ? at : kOut, 0, 0),
                                            __builtin_amdgcn_raw_buffer_load_b32(rs, left > 2 ? at + 4 : kOut, 0, 0)});
  bf16x4 v;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    v[k] = __builtin_bit_cast(__bf16, __builtin_amdgcn_raw_buffer_load_b16(rs, left > k ? at + 2 * k : kOut, 0, 0));
  return v;
}
__device__ __forceinline__ f32x4 wide(bf16x4 v) { return f32x4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]}; }

// The gradients of a chunk but dV, from bf16 inputs: eight waves, one workgroup a
// CU.  Waves 0-3 (`reader`) and 4-7 share the work by what it is about:
//   1  16 columns of v a wave: Y from S, and R from D, as in the walks; their parts
//      go to LDS by rows
//   2  16 tokens a wave, all products transposed, so that a result of 16 tokens'
//      columns is the second operand of the next as it stands.  A reader's tokens
//      are i: S dO^T and S R^T for dQ and dKr, (Y dO^T)_ji and (Y R^T)_ji; the
//      others' are j: D Y^T for dKw, (dO Y^T)_ij and (R Y^T)_ij
//   3  the latter, with their factors dP o M = scale beta_j M_ij dO Y^T and
//      dL o M = -beta_i beta_j M_ij R Y^T, times K, Q and K
// dbeta is the diagonal of Y R^T.  Tile rows left of the diagonal for a reader are
// right of it for its partner on the same SIMD, so the SIMDs' work is even.
// LDS: K by rows, then columns; dO; Q by rows, then Y and R, then C and dKw; Z,
// its transpose and P's, then S and D (one after the other for more than 64 rows)
// and Q by columns.  ONE: dv <= 64, so that what part 2 adds up need not live
// through part 1.  Where it does, 94, 172, 229 and 334 registers spill for KS = 1 to 4:
// 2048 chunks of dv = 64 take 170 us with ONE and 386 without for dk = 64, 227 and 708
// for dk = 128, and of dv = 128, which has two slices, 262, 388 and 717 for dk = 32, 64,
// 128.
// What bounds it: 2048 chunks of d = 64 take 166 us, where their bytes take 37.  With
// one workgroup a CU nothing covers a chunk's first loads (a fifth of its 41000
// cycles) and the waits at the nine barriers; the two waves of a SIMD issue vector
// instructions two fifths of the time.  Tried without gain: workgroups that go
// through several chunks and load the next one ahead (the registers for it spill).
template <int KS, bool ONE>
__global__ void __launch_bounds__(512, 2) delta_grads_parts_kernel(const DeltaParams p) {
  typedef __bf16 T;
  constexpr int NT = 512, DK = 32 * KS, LDK = DK + 8, L = 72, ST = 2 * KS;
  constexpr int kK = 64 * LDK, kKt = DK * L, kVal = 64 * L, kState = DK * L, LW = DK + 4;
  constexpr bool kBoth = KS <= 2;
  constexpr int kFirst = kK > kKt ? kK : kKt;
  constexpr int kStates = (kBoth ? 6 : 3) * kState, kLast = 9 * kTri > kStates + kKt ? 9 * kTri : kStates + kKt;
  static_assert(kK <= 6 * kVal && 2 * (kTile + 64 * LW) <= 6 * kVal, "Q, or C and dKw, fit the place of Y and R");
  __shared__ __attribute__((aligned(16))) unsigned short first[kFirst], yr[7 * kVal], rest[kLast];
  __shared__ __attribute__((aligned(16))) float gt[kGateFloats];
  __shared__ float pairs[8][64], part[8], reads[64], writes[64], dbeta[64];
  unsigned short* const os = yr + 6 * kVal;
  unsigned short *const zp = rest, *const zt = rest + 3 * kTri, *const pt = rest + 6 * kTri;
  unsigned short *const sp = rest, *const dp = rest + (kBoth ? 3 * kState : 0), *const qt = rest + kStates;
  float *const cs = reinterpret_cast<float*>(yr), *const ws = cs + kTile;
  const int64_t chunk = blockIdx.x;
  const At w = chunk_at(p, chunk);
  const int tid = threadIdx.x, wave = tid >> 6, st = wave & 3, l = tid & 63, r = l & 15, g = l >> 4;
  const bool reader = wave < 4;
  const int tok = 16 * st + r;                          // the token of this lane in parts 2 and 3
  const int hk = w.h / (p.H / p.Hk);
  const bool shared_heads = p.H != p.Hk;                // dq and dk are then fp32, by head
  const int rows = (int)min((int64_t)kDeltaChunk, p.S - w.t0);
  auto put_qk = [&](const DeltaRows& dst, int row, int col, f32x4 v) {
    const int left = p.dk_ - col;
    if (shared_heads) {
      float* const o = row_ptr<float>(dst, w.b, w.t0 + row, w.h) + col;
      if (p.out_vec) {
        if (left > 0) store4(o, v);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (k < left) o[k] = v[k];
      }
    } else {
      T* const o = row_ptr<T>(dst, w.b, w.t0 + row, w.h) + col;
      const bf16x4 n = __builtin_convertvector(v, bf16x4);
      if (p.out_vec) {
        if (left > 0) *reinterpret_cast<bf16x4*>(o) = n;
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (k < left) o[k] = n[k];
      }
    }
  };
  auto put_gate = [&](const DeltaRows& dst, int row, float v) { *row_ptr<float>(dst, w.b, w.t0 + row, w.h) = v; };
  if (w.rows == 0) {
    for (int row = wave; row < rows; row += 8) {
      for (int e = 4 * l; e < p.dk_; e += 256) {
        put_qk(p.dq, row, e, zero4());
        put_qk(p.dk, row, e, zero4());
      }
      if (l == 0) {
        put_gate(p.dg, row, 0.0f);
        put_gate(p.dbeta, row, 0.0f);
      }
    }
    return;
  }
  const T* const q = row_ptr<T>(p.q, w.b, w.t0, hk);
  const T* const k = row_ptr<T>(p.k, w.b, w.t0, hk);
  const T* const v = row_ptr<T>(p.v, w.b, w.t0, w.h);
  const T* const go = row_ptr<T>(p.dout, w.b, w.t0, w.h);
  const float* const sg = p.s + chunk * DK * p.dvp;
  const float* const dg = p.d + chunk * DK * p.dvp;
  const Rsrc o_rs = rows_rsrc<T>(go, p.dout.ss, w.rows, p.dv_);
  const Rsrc raw_rs = reader ? rows_rsrc<T>(v, p.v.ss, w.rows, p.dv_) : o_rs;
  const unsigned raw_row = 2u * (unsigned)(reader ? p.v.ss : p.dout.ss);
  const Rsrc state_rs = make_rsrc(reader ? sg : dg, (unsigned)DK * p.dvp * 4u);
  const int zi = tid < 64 ? 4 * (tid >> 3) : 32 + 4 * ((tid - 64) >> 4), zj = 4 * (tid < 64 ? tid & 7 : (tid - 64) & 15);
  Block<T, KS, NT> kb, qb;
  kb.load(k, p.k.ss, w.rows, p.dk_, p.vec);
  qb.load(q, p.q.ss, w.rows, p.dk_, p.vec);
  for (int e = tid; e < kGateFloats; e += NT) gt[e] = p.gates[chunk * kGateFloats + e];
  f32x4 a1[ST], a2[ST];                 // dQ^T and dKr^T, or dKw^T and nothing
  f32x4 mp[4], ml[4], qk[4], kk[4];     // dO Y^T, R Y^T, and a reader's K Q^T, K K^T, by tiles of the other token
  if (!ONE) {
    clear(a1);
    clear(a2);
    clear(mp);
    clear(ml);
  }
  // K and Q for part 3, and the rows of this lane's token as its results lie
  const Rsrc k_rs = rows_rsrc<T>(k, p.k.ss, w.rows, p.dk_), q_rs = rows_rsrc<T>(q, p.q.ss, w.rows, p.dk_);
  bf16x4 k_tok[ST], q_tok[ST];
  auto load_tokens = [&] {
    kb.load(k, p.k.ss, w.rows, p.dk_, p.vec);
    qb.load(q, p.q.ss, w.rows, p.dk_, p.vec);
#pragma unroll
    for (int t = 0; t < ST; ++t) {
      const int c = 16 * t + 4 * g;
      k_tok[t] = load_quad(k_rs, tok * 2u * (unsigned)p.k.ss + 2 * c, p.dk_ - c, p.vec);
      if (reader) q_tok[t] = load_quad(q_rs, tok * 2u * (unsigned)p.q.ss + 2 * c, p.dk_ - c, p.vec);
    }
  };
  float ending = 0.0f;
  for (int vb = 0; vb < (ONE ? 1 : p.dvp); vb += 64) {
    if (vb) {
      __syncthreads();
      qb.load(q, p.q.ss, w.rows, p.dk_, p.vec);
    }
    // the slice's inputs
    const int col = vb + 16 * st + r;
    f32x4 state[ST];
    unsigned raw[16];
#pragma unroll
    for (int t = 0; t < ST; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        state[t][i] = raw_value<float>(load_raw<float>(state_rs, col < p.dvp ? (unsigned)((16 * t + 4 * g + i) * p.dvp + col) * 4u : kOut));
    const unsigned raw_at = col < p.dv_ ? 2u * col + 4 * g * raw_row : kOut;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) raw[4 * t + i] = load_raw<T>(raw_rs, raw_at, (16 * t + i) * raw_row);
    bf16x4 oq[2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int e = tid + n * NT, c = vb + 4 * (e & 15);
      oq[n] = load_quad(o_rs, (e >> 4) * 2u * (unsigned)p.dout.ss + 2u * c, p.dv_ - c, p.vec);
    }
    f32x4 zr[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = min(zi, 60) + i, quad = row < 32 ? row * 8 + (zj >> 2) : 256 + (row - 32) * 16 + (zj >> 2);
      zr[i] = load4(p.z + chunk * kZFloats + 4 * quad);
    }
    if (vb == 0) kb.template put_rows<LDK>(first, kFirst);   // (when all loads are on their way)
    qb.template put_rows<LDK>(yr, kK);
#pragma unroll
    for (int n = 0; n < 2; ++n) *reinterpret_cast<bf16x4*>(os + ((tid + n * NT) >> 4) * L + 4 * ((tid + n * NT) & 15)) = oq[n];
    __syncthreads();
    if (tid < 192) {
      const f32x4 beta = load4(gt + kBeta + zj);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        u32x2 parts[3];
        split4<3>(parts, -zr[i] * beta);      // -Z beta
#pragma unroll
        for (int n = 0; n < 3; ++n) *reinterpret_cast<u32x2*>(zp + n * kTri + tri_at(zi + i) + place4(zj >> 2)) = parts[n];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) zr[i] *= -gt[kBeta + zi + i];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        u32x2 parts[3];
        split4<3>(parts, f32x4{zr[0][j], zr[1][j], zr[2][j], zr[3][j]});   // -(beta Z)^T
#pragma unroll
        for (int n = 0; n < 3; ++n) *reinterpret_cast<u32x2*>(zt + n * kTri + upper_at(zj + j, place4(zi >> 2))) = parts[n];
      }
    }
    if (reader) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        qk[t] = kk[t] = zero4();
        if (t <= st)
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            u32x4 a[1], bq[1], bk[1];
            read_parts<1>(a, first, 0, (16 * t + r) * LDK + 32 * s + 8 * g);
            read_parts<1>(bq, yr, 0, tok * LDK + 32 * s + 8 * g);
            read_parts<1>(bk, first, 0, tok * LDK + 32 * s + 8 * g);
            qk[t] = mfma(a[0], bq[0], qk[t]);
            kk[t] = mfma(a[0], bk[0], kk[t]);
          }
      }
    } else {
      // scale P^T: ten tiles and the two of zeros that complete their pairs, three a wave
#pragma unroll
      for (int e = 0; e < 3; ++e) {
        const int tr = e < 2 ? e : 2 + (st >> 1), t = e < 2 ? st : 2 + (st & 1), row = 16 * tr + r;
        f32x4 acc = zero4();
        if (t >= tr) {
          u32x4 a[KS][1], bk[KS][1];
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            read_parts<1>(a[s], yr, 0, (16 * t + r) * LDK + 32 * s + 8 * g);
            read_parts<1>(bk[s], first, 0, row * LDK + 32 * s + 8 * g);
          }
#pragma unroll
          for (int s = 0; s < KS; ++s) acc = mfma(a[s][0], bk[s][0], acc);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int q_row = 16 * t + 4 * g + i;
            acc[i] = q_row >= row ? p.scale * acc[i] * decay(gt, q_row, row) : 0.0f;
          }
        }
        u32x2 parts[3];
        split4<3>(parts, acc);
#pragma unroll
        for (int n = 0; n < 3; ++n) *reinterpret_cast<u32x2*>(pt + n * kTri + upper_at(row, place4(4 * t + g))) = parts[n];
      }
    }
    __syncthreads();
    // the states of part 2 on their way
    constexpr int NS = DK * 16 / NT;   // quads a thread
    f32x4 sq[NS], dq[NS];
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      const int e = tid + n * NT, c = vb + 4 * (e & 15);
      const int64_t at = (int64_t)(e >> 4) * p.dvp + c;
      sq[n] = c < p.dvp ? load4(sg + at) : zero4();
      dq[n] = c < p.dvp ? load4(dg + at) : zero4();
    }
    // 1
    {
      f32x4 x[4];
      clear(x);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        u32x4 b[3];
        split_pair<3>(b, state[2 * s], state[2 * s + 1]);
        products<1, 3, 4>(
            0, [&](int i) { return first + (16 * i + r) * LDK + 32 * s + 8 * g; },
            [&](int i, const u32x4(&a)[1]) { mul<3, 2>(x[i], a, b); });
      }
      u32x4 xp[2][3];
      if (reader) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const f32x4 gam = load4(gt + kGam + 16 * t + 4 * g);
#pragma unroll
          for (int i = 0; i < 4; ++i) x[t][i] = raw_value<T>(raw[4 * t + i]) - gam[i] * x[t][i];
        }
        split_pair<3>(xp[0], x[0], x[1]);
        split_pair<3>(xp[1], x[2], x[3]);
        products<3, 1, 6>(
            kTri, [&](int i) { return zp + tri_at(16 * (i < 4 ? i : i - 2) + r) + 32 * (i >> 2) + 8 * g; },
            [&](int i, const u32x4(&a)[3]) { mul<3, 2>(x[i < 4 ? i : i - 2], a, xp[i >> 2]); });
      } else {
        u32x4 ob[2][1];
#pragma unroll
        for (int s = 0; s < 2; ++s)
          ob[s][0] = u32x4{raw[8 * s] | raw[8 * s + 1] << 16, raw[8 * s + 2] | raw[8 * s + 3] << 16,
                           raw[8 * s + 4] | raw[8 * s + 5] << 16, raw[8 * s + 6] | raw[8 * s + 7] << 16};
#pragma unroll
        for (int t = 0; t < 4; ++t) x[t] *= load4(gt + kEnd + 16 * t + 4 * g);
        products<3, 1, 6>(
            kTri, [&](int i) { return pt + upper_at(16 * (i < 2 ? i : i - 2) + r, 32 * (i >= 2) + 8 * g); },
            [&](int i, const u32x4(&a)[3]) { mul<1, 2>(x[i < 2 ? i : i - 2], a, ob[i >= 2]); });
        split_pair<3>(xp[0], x[0], x[1]);
        split_pair<3>(xp[1], x[2], x[3]);
        products<3, 1, 6>(
            kTri, [&](int i) { return zt + upper_at(16 * (i < 2 ? i : i - 2) + r, 32 * (i >= 2) + 8 * g); },
            [&](int i, const u32x4(&a)[3]) { mul<3, 2>(x[i < 2 ? i : i - 2], a, xp[i >= 2]); });
      }
      // (columns past dv are zeros: the states' padding, v and dO are)
      unsigned short* const dst = yr + (reader ? 0 : 3 * kVal) + 16 * st + r;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        u32x2 parts[3];
        split4<3>(parts, x[t]);
#pragma unroll
        for (int n = 0; n < 3; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            dst[n * kVal + (16 * t + 4 * g + i) * L] = (unsigned short)(parts[n][i >> 1] >> (16 * (i & 1)));
      }
    }
    __syncthreads();
    auto put_state = [&](unsigned short* to, const f32x4(&from)[NS]) {
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        const int e = tid + n * NT;
        u32x2 parts[3];
        split4<3>(parts, from[n]);
#pragma unroll
        for (int m = 0; m < 3; ++m) *reinterpret_cast<u32x2*>(to + m * kState + (e >> 4) * L + 4 * (e & 15)) = parts[m];
      }
    };
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) ending = __builtin_fmaf(sq[n][i], dq[n][i], ending);
    put_state(sp, sq);
    if (kBoth) put_state(dp, dq);
    __syncthreads();
    // 2
    if (ONE) {
      clear(a1);
      clear(a2);
      clear(mp);
      clear(ml);
      if (kBoth) load_tokens();   // for part 3, where registers allow it
    }
    const unsigned short *const ys = yr, *const rs = yr + 3 * kVal;
    u32x4 bo[2][1], b3[2][3];   // the tokens' dO and R, or Y
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      read_parts<1>(bo[s], os, 0, tok * L + 32 * s + 8 * g);
      read_parts<3>(b3[s], reader ? rs : ys, kVal, tok * L + 32 * s + 8 * g);
    }
    auto by_states = [&] {
      if (reader)
        products<3, 1, 2 * ST>(
            kState, [&](int i) { return sp + (16 * (i >> 1) + r) * L + 32 * (i & 1) + 8 * g; },
            [&](int i, const u32x4(&a)[3]) {
              mul<1, 2>(a1[i >> 1], a, bo[i & 1]);
              mul<3, 2>(a2[i >> 1], a, b3[i & 1]);
            });
    };
    auto by_gradients = [&] {
      if (!reader)
        products<3, 1, 2 * ST>(
            kState, [&](int i) { return dp + (16 * (i >> 1) + r) * L + 32 * (i & 1) + 8 * g; },
            [&](int i, const u32x4(&a)[3]) { mul<3, 2>(a1[i >> 1], a, b3[i & 1]); });
    };
    auto by_tokens = [&] {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        if (reader ? t > st : t < st) continue;
        const int at = (16 * t + r) * L + 8 * g;
        if (reader) {
          products<3, 1, 2>(
              kVal, [&](int i) { return ys + at + 32 * i; },
              [&](int i, const u32x4(&a)[3]) {
                mul<1, 2>(mp[t], a, bo[i]);
                mul<3, 2>(ml[t], a, b3[i]);
              });
        } else {
          products<4, 1, 2>(   // R's parts and dO after them
              kVal, [&](int i) { return rs + at + 32 * i; },
              [&](int i, const u32x4(&a)[4]) {
                const u32x4 ar[3] = {a[0], a[1], a[2]}, ao[1] = {a[3]};
                mul<3, 2>(ml[t], ar, b3[i]);
                mul<3, 2>(mp[t], ao, b3[i]);
              });
        }
      }
    };
    by_states();
    if (kBoth) {
      by_gradients();
      by_tokens();
    } else {
      if (!reader) by_tokens();
      __syncthreads();
      put_state(dp, dq);
      __syncthreads();
      by_gradients();
      if (reader) by_tokens();
    }
  }
  if (!ONE || !kBoth) load_tokens();
  __syncthreads();
  kb.template put_columns<L>(first, kFirst);
  qb.template put_columns<L>(qt, kKt);
  // the factors of this lane's token, and the gates' parts of what S and D gave
  const float gam = gt[kGam + tok], beta = gt[kBeta + tok];
  float dot = 0.0f;
  {
    const float f1 = reader ? p.scale * gam : gt[kEnd + tok] * beta, f2 = -gam * beta;
#pragma unroll
    for (int t = 0; t < ST; ++t) {
      const f32x4 kv = wide(k_tok[t]);
      a1[t] *= f1;
      if (reader) {
        const f32x4 qv = wide(q_tok[t]);
        a2[t] *= f2;
#pragma unroll
        for (int i = 0; i < 4; ++i) dot += qv[i] * a1[t][i] + kv[i] * a2[t][i];
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) dot = __builtin_fmaf(kv[i], a1[t][i], dot);
      }
    }
    dot += __shfl_xor(dot, 16);
    dot += __shfl_xor(dot, 32);
    if (g == 0) (reader ? reads : writes)[tok] = dot;
  }
  // dP o M and dL o M, their pairs' part of dg, dbeta
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const f32x4 bo = load4(gt + kBeta + 16 * t + 4 * g);
    f32x4 c = zero4();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int other = 16 * t + 4 * g + i, ri = reader ? tok : other, cj = reader ? other : tok;
      if (reader && other == tok) dbeta[tok] = ml[t][i];
      const float m = ri >= cj ? decay(gt, ri, cj) : 0.0f;
      mp[t][i] = ri >= cj ? p.scale * (reader ? bo[i] : beta) * m * mp[t][i] : 0.0f;
      ml[t][i] = ri > cj ? -beta * bo[i] * m * ml[t][i] : 0.0f;
      if (reader && ri > cj) c[i] = mp[t][i] * qk[t][i] + ml[t][i] * kk[t][i];
    }
    if (reader) *reinterpret_cast<f32x4*>(cs + tok * kLd + 16 * t + 4 * g) = c;
  }
  __syncthreads();
  // 3
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    if (reader ? 2 * s > st : 2 * s + 1 < st) continue;
    u32x4 bp[3], bl[3];
    split_pair<3>(bp, mp[2 * s], mp[2 * s + 1]);
    split_pair<3>(bl, ml[2 * s], ml[2 * s + 1]);
    if (reader)
      products<1, 2, ST>(
          0, [&](int i) { return first + (16 * i + r) * L + 32 * s + 8 * g; },
          [&](int i, const u32x4(&a)[1]) {
            mul<3, 2>(a1[i], a, bp);
            mul<3, 2>(a2[i], a, bl);
          });
    else
      products<1, 2, 2 * ST>(
          0, [&](int i) { return (i < ST ? qt : first) + (16 * (i % ST) + r) * L + 32 * s + 8 * g; },
          [&](int i, const u32x4(&a)[1]) { mul<3, 2>(a1[i % ST], a, i < ST ? bp : bl); });
  }
  if (!reader)
#pragma unroll
    for (int t = 0; t < ST; ++t) *reinterpret_cast<f32x4*>(ws + tok * LW + 16 * t + 4 * g) = a1[t];
  {
    // C over its rows i in [8 wave, 8 wave + 8) for every t, lane t: over j < t by a
    // scan along the row, then over the rows at and past t.
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int row = 8 * wave + i;
      float c = cs[row * kLd + l];
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const float up = __shfl_up(c, o);
        if (l >= o) c += up;
      }
      const float before = __shfl_up(c, 1);   // sum_{j < t}
      if (l > 0 && row >= l) sum += before;
    }
    pairs[wave][l] = sum;
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) ending += __shfl_xor(ending, o);
  if (l == 0) part[wave] = ending;
  __syncthreads();
  if (reader && tok < rows)
#pragma unroll
    for (int t = 0; t < ST; ++t) {
      const int c = 16 * t + 4 * g;
      put_qk(p.dq, tok, c, a1[t]);
      put_qk(p.dk, tok, c, a2[t] + *reinterpret_cast<const f32x4*>(ws + tok * LW + c));
    }
  if (wave == 7) {
    float from = reads[l], upto = writes[l];
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const float down = __shfl_down(from, o), up = __shfl_up(upto, o);
      if (l + o < 64) from += down;
      if (l >= o) upto += up;
    }
    upto = __shfl_up(upto, 1);
    float sum = from + (l > 0 ? upto : 0.0f), whole = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      sum += pairs[i][l];
      whole += part[i];
    }
    if (l < rows) {
      put_gate(p.dg, l, l < w.rows ? sum + gt[kGam + 63] * whole : 0.0f);
      put_gate(p.dbeta, l, l < w.rows ? dbeta[l] : 0.0f);
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

template <typename T, int KS>
hipError_t walks(const DeltaParams& p, hipStream_t stream) {
  if (p.segs > 1) {
    launch_rewalk<T, KS, true>(p, stream);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess)
      e = launch_delta_scan(p, p.a, p.x, p.grad_state, p.segs, p.seg * kDeltaChunk, true, stream);
    if (e != hipSuccess) return e;
  }
  launch_rewalk<T, KS, false>(p, stream);
  return hipGetLastError();
}

template <typename T>
hipError_t backward(const DeltaParams& p, float* const part, hipStream_t stream) {
  const unsigned chunks = (unsigned)((int64_t)p.B * p.H * p.N);
  hipError_t e;
  switch (p.dkp / 32) {
    case 1: e = walks<T, 1>(p, stream); break;
    case 2: e = walks<T, 2>(p, stream); break;
    case 3: e = walks<T, 3>(p, stream); break;
    default: e = walks<T, 4>(p, stream); break;
  }
  if (e != hipSuccess) return e;
  const int64_t plane = (int64_t)p.B * p.S * p.H * p.dk_;
  DeltaParams w = p;
  if (p.H != p.Hk) {
    const DeltaRows own = {nullptr, (int64_t)p.S * p.H * p.dk_, (int64_t)p.H * p.dk_, p.dk_};
    w.dq = w.dk = own;
    w.dq.p = part;
    w.dk.p = part + plane;
  }
  if constexpr (sizeof(T) == 2) {
    auto go = [&](auto ks) {
      constexpr int KS = decltype(ks)::value;
      if (p.dvp <= 64)
        hipLaunchKernelGGL((delta_grads_parts_kernel<KS, true>), dim3(chunks), dim3(512), 0, stream, w);
      else
        hipLaunchKernelGGL((delta_grads_parts_kernel<KS, false>), dim3(chunks), dim3(512), 0, stream, w);
    };
    switch (p.dkp / 32) {
      case 1: go(std::integral_constant<int, 1>{}); break;
      case 2: go(std::integral_constant<int, 2>{}); break;
      case 3: go(std::integral_constant<int, 3>{}); break;
      default: go(std::integral_constant<int, 4>{}); break;
    }
  } else if (p.dkp <= 64) {
    hipLaunchKernelGGL((delta_grads_kernel<1>), dim3(chunks), dim3(kGradThreads), 0, stream, w);
  } else {
    hipLaunchKernelGGL((delta_grads_kernel<2>), dim3(chunks), dim3(kGradThreads), 0, stream, w);
  }
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
