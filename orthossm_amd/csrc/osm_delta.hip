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
//   S' = e^{G_last} S + K^T (e^{G_last - G} U)
// Every column of S (and of V, X, U, O) goes its own way.
//
// Launches:
//   solve   Z and the gates of every chunk at once.
//   walk    a workgroup walks a segment of a row's chunks, each wave 16 columns
//           of S in its accumulators.  The accumulator of one product is the
//           second operand of the next as it stands (its rows are the terms of
//           the sum), so X, U and S never leave the registers; K, Q, Z and P, the
//           first operands, are shared by the waves through LDS.
// Where the rows and heads alone do not fill the chip, rows are cut into
// segments: a first walk from zero and from the columns of the identity gives
// every segment's affine map of the state, `scan` joins them, and the second
// walk gives the outputs from the right states.
//
// Products run on the bf16 matrix instruction at fp32's accuracy: an fp32 operand
// is the sum of three bf16 numbers (8 bits each; the remainders are exact), bf16
// inputs are one, and of the products of parts those of order 2^-24 and below are
// left out: 3 instructions against a bf16 operand, 6 between two fp32 ones, where
// the fp32 matrix instruction takes 16 times as long as the bf16 one.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "osm_delta.h"

namespace osm {
namespace {

using namespace delta;

// Z from L in place (tile zs, L strictly lower, zeros elsewhere), by one wave: the
// four diagonal 16x16 blocks by substitution, row i from the rows before it (Z_i
// = L_i - sum_j L_ij beta_j Z_j), then block pairs: for L = [[a, 0], [c, d]],
// Z_c = (I - Z_d beta) (L_c - L_c beta Z_a), the 16-wide ones, then the 32-wide.
__device__ __forceinline__ void invert(float* zs, const float* beta) {
  const int l = threadIdx.x & 63, c = l & 15, o = 16 * (l >> 4);
  float* const base = zs + o * kLd + o;
  float z[16], bz[16];   // column c of the lane's block of Z, and beta Z
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float v = base[i * kLd + c];
    f32x4 row[4];
#pragma unroll
    for (int q = 0; q < (i + 3) / 4; ++q) row[q] = load4(base + i * kLd + 4 * q);
#pragma unroll
    for (int j = 0; j < i; ++j) v = __builtin_fmaf(-row[j / 4][j % 4], bz[j], v);
    z[i] = v;
    bz[i] = beta[o + i] * v;
  }
  __syncthreads();   // (one wave: orders its lanes' accesses)
#pragma unroll
  for (int i = 0; i < 16; ++i) base[i * kLd + c] = z[i];
  __syncthreads();
  f32x4 acc[2][1], q[2][1];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int a = 32 * h, d = a + 16;
    clear(acc[h]);
    mma<1, false, false, true>(acc[h], zs, d, zs, a, a, d, beta);   // L_c beta Z_a
    get(q[h], zs, d, a);
    q[h][0] -= acc[h][0];
  }
  __syncthreads();
  put(zs, q[0], 16, 0);
  put(zs, q[1], 48, 32);
  __syncthreads();
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int a = 32 * h, d = a + 16;
    clear(acc[h]);
    mma<1, false, false, true>(acc[h], zs, d, zs, a, d, d + 16, beta);   // Z_d beta (..)
    q[h][0] -= acc[h][0];
  }
  __syncthreads();
  put(zs, q[0], 16, 0);
  put(zs, q[1], 48, 32);
  __syncthreads();
  f32x4 wide[2][2], w[2][2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    clear(wide[h]);
    mma<2, false, false, true>(wide[h], zs, 32 + 16 * h, zs, 0, 0, 32, beta);
    get(w[h], zs, 32 + 16 * h, 0);
    w[h][0] -= wide[h][0];
    w[h][1] -= wide[h][1];
  }
  __syncthreads();
  put(zs, w[0], 32, 0);
  put(zs, w[1], 48, 0);
  __syncthreads();
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    clear(wide[h]);
    mma<2, false, false, true>(wide[h], zs, 32 + 16 * h, zs, 0, 32, 64, beta);
    w[h][0] -= wide[h][0];
    w[h][1] -= wide[h][1];
  }
  __syncthreads();
  put(zs, w[0], 32, 0);
  put(zs, w[1], 48, 0);
  __syncthreads();
}

// Z and the gates of a chunk, one wave: the steps of the inversion follow each
// other closely and hold little, so eight chunks a CU side by side beat four waves
// that wait for each other (8192 chunks of d = 64: 89 us with four waves, 59 so).
// What bounds it: the chain of the substitution and of the block products, a third
// of its time waiting for LDS.  KS: blocks of 32 columns of k.
template <typename T, int KS>
__global__ void __launch_bounds__(64) delta_solve_kernel(const DeltaParams p) {
  constexpr int NP = kParts<T>, LDK = 32 * KS + 8, kBytes = NP * 64 * LDK * 2 > 4 * kTile ? NP * 64 * LDK * 2 : 4 * kTile;
  __shared__ __attribute__((aligned(16))) unsigned char both[kBytes];   // K, then L and Z
  __shared__ __attribute__((aligned(16))) float gt[kGateFloats];
  unsigned short* const kk = reinterpret_cast<unsigned short*>(both);
  float* const zs = reinterpret_cast<float*>(both);
  const int64_t chunk = blockIdx.x;
  const At w = chunk_at(p, chunk);
  if (w.rows == 0) return;
  const int l = threadIdx.x, r = l & 15, g = l >> 4;
  Block<T, KS, 64> kb;
  kb.load(row_ptr<T>(p.k, w.b, w.t0, w.h / (p.H / p.Hk)), p.k.ss, w.rows, p.dk_, p.vec);
  make_gates(gt, p.g, p.beta, w.b, w.t0, w.h, w.rows);
  kb.template put_rows<LDK>(kk, 64 * LDK);
  __syncthreads();
  f32x4 acc[4][4];   // [c][t]: element i is (K K^T)[16 c + 4 g + i][16 t + r], for c <= t
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    clear(acc[t]);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      u32x4 b[NP];
      read_parts<NP>(b, kk, 64 * LDK, (16 * t + r) * LDK + 32 * s + 8 * g);
#pragma unroll
      for (int c = 0; c <= t; ++c) {
        u32x4 a[NP];
        read_parts<NP>(a, kk, 64 * LDK, (16 * c + r) * LDK + 32 * s + 8 * g);
        mul<NP, 2>(acc[t][c], a, b);
      }
    }
  }
  __syncthreads();
  // (it is symmetric: four columns of row 16 t + r a lane)
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int row = 16 * t + r, col = 16 * c + 4 * g;
      f32x4 v = zero4();
      if (c <= t)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = row > col + i ? acc[t][c][i] * decay(gt, row, col + i) : 0.0f;
      *reinterpret_cast<f32x4*>(zs + row * kLd + col) = v;
    }
  __syncthreads();
  invert(zs, gt + kBeta);
  float* const zg = p.z + chunk * kZFloats;
#pragma unroll
  for (int e = l; e < kZFloats / 4; e += 64)
    store4(zg + 4 * e, *reinterpret_cast<const f32x4*>(zs + z_row(e) * kLd + 4 * z_quad(e)));
  float* const gg = p.gates + chunk * kGateFloats;
#pragma unroll
  for (int e = l; e < kGateFloats; e += 64) gg[e] = gt[e];
}

// S' = A S + B over the spans of a row, in order or in reverse, for 16 columns
// of S: wave w holds rows 16 w .. 16 w + 15 of S and of A, and S passes between
// the waves through LDS, transposed ([column][row], so that both the
// accumulators' four rows and the product's four terms are one 16-byte access),
// in two buffers: one barrier a span.  x holds B and receives the state before
// the span.  KT = dkp / 16.  What bounds it: the chain of spans, 4 KT matrix
// instructions and the exchange each (32 spans of 16 heads, dk = dv = 64: 15 us;
// maps read three spans ahead instead of one: 18).
template <int KT>
__global__ void __launch_bounds__(64 * KT) delta_scan_kernel(const float* a, float* x, const float* init,
                                                             const int* lengths, int S, int N, int span, int BH, int H,
                                                             int dk, int dv, int dvp, bool reverse) {
  constexpr int kDkp = 16 * KT, kRow = kDkp + 4;
  __shared__ __attribute__((aligned(16))) float st[2][16 * kRow];
  // The column slices of a head share A, so they take one XCD (workgroups go
  // round the eight XCDs by their index).
  const int ns = dvp / kDeltaSlice, j = blockIdx.x >> 3, bh = (j / ns) * 8 + (blockIdx.x & 7);
  if (bh >= BH) return;
  const int wave = threadIdx.x >> 6, l = threadIdx.x & 63, r = l & 15, g = l >> 4;
  const int col = kDeltaSlice * (j % ns) + r, row = 16 * wave + 4 * g;
  const int tokens = lengths ? min(max(lengths[bh / H], 0), S) : S;
  const int n = (int)(((int64_t)tokens + span - 1) / span);
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
  if (n > 1) fetch(0);
  for (int c = 0; c < n; ++c) {
    float* const xp = x + at(c) * kDkp * dvp;
    if (c == n - 1) {   // the last span's map is not needed
#pragma unroll
      for (int i = 0; i < 4; ++i) xp[(int64_t)i * dvp] = s[i];
      break;
    }
    float* const buf = st[c & 1];
    *reinterpret_cast<f32x4*>(buf + r * kRow + row) = s;
    f32x4 ac[KT], acc0 = bn, acc1 = zero4();
#pragma unroll
    for (int k = 0; k < KT; ++k) ac[k] = an[k];
    if (c + 2 < n) fetch(c + 1);
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
}

// Walks segment blockIdx.x % segs of a head.  MAP: the segment's state map, from
// zero for the columns of v and from the identity's columns after them; else the
// outputs.  KS: blocks of 32 rows of S; WAVES: of 16 columns each.
// What bounds it: 256 chunks of 32 heads, bf16, d = 64, take 134 us for the maps and
// 138 for the outputs, in which the vector instructions (the parts of X, U, S, Z, P)
// fill a third of the time, the matrix instructions a quarter, LDS two fifths, and
// the two or three waves a SIMD has room for wait for each other in between.  fp32
// outputs take 101 KB of LDS (d = 64): four waves a CU, one a SIMD (three rows of up to
// 5001 tokens, 8 heads, d = 50: 71 us, the maps at two waves a SIMD 46).  Tried without gain: products of two tiles in turn, a higher priority for
// waves in their products, 128 registers for twice the waves, and LDS rows 160 bytes
// apart, whose 16-byte reads meet no bank twice (their writes meet more: 144 us).
template <typename T, int KS, int WAVES, bool MAP>
__global__ void __launch_bounds__(64 * WAVES, 2) delta_walk_kernel(const DeltaParams p, int groups) {
  constexpr int NT = 64 * WAVES, NP = kParts<T>, DK = 32 * KS, LDK = DK + 8, LKT = 72, ST = 2 * KS;
  // By parts: K by rows, K by columns, Q by rows; where two workgroups' LDS does not
  // hold all three, Q first has the place of K by columns.  Then Z and P.
  constexpr int kK = 64 * LDK, kKt = DK * LKT;
  constexpr bool kApart = !MAP && 2 * (NP * (kKt + 2 * kK) + 6 * kTri) + 8 * kGateFloats <= 80 * 1024;
  constexpr int kIn = kK + (MAP ? kKt : kApart ? kKt + kK : kKt > kK ? kKt : kK);
  __shared__ __attribute__((aligned(16))) unsigned short in[NP][kIn], zp[3][kTri], pp[MAP ? 1 : 3][MAP ? 8 : kTri];
  __shared__ __attribute__((aligned(16))) float gates[2][kGateFloats];
  unsigned short *const kk = &in[0][0], *const kt = kk + kK, *const qq = kApart ? kt + kKt : kt;
  const int group = blockIdx.x % groups;
  const int64_t id = blockIdx.x / groups;
  const int seg = (int)(id % p.segs), bh = (int)(id / p.segs), b = bh / p.H, h = bh - b * p.H, hk = h / (p.H / p.Hk);
  const int tid = threadIdx.x, wave = tid >> 6, l = tid & 63, r = l & 15, g = l >> 4;
  const int tokens = p.lengths ? min(max(p.lengths[b], 0), p.S) : p.S;
  const int n = (tokens + kDeltaChunk - 1) / kDeltaChunk;          // chunks in use
  const int c0 = seg * p.seg, c1 = min(min(c0 + p.seg, p.N), n);
  const int slice = group * WAVES + wave, vs = p.dvp / kDeltaSlice;
  const bool value = slice < vs, live = slice < vs + (MAP ? DK / kDeltaSlice : 0);
  const int col = kDeltaSlice * slice + r;                         // of v, or dvp + of the identity
  const bool in_v = value && col < p.dv_;
  if (!MAP) {
    // zeros for the chunks without tokens
    for (int c = max(c0, n); c < min(c0 + p.seg, p.N); ++c) {
      T* const o = row_ptr<T>(p.o, b, (int64_t)c * kDeltaChunk, h) + col;
      if (in_v)
        for (int t = g; t < min(kDeltaChunk, p.S - c * kDeltaChunk); t += 4) o[t * p.o.ss] = (T)0.0f;
    }
  }
  const bool fin = !MAP && p.fin && seg == (n > 0 ? (n - 1) / p.seg : 0);
  if (c0 >= c1 && !fin) return;
  if (MAP && c1 == n) return;   // nothing follows the last segment
  // S: tile t, element i: row 16 t + 4 g + i, column col
  f32x4 S[ST];
  const bool ws = !MAP && p.segs > 1 && n > 0;
  const float* const from = MAP ? nullptr : ws ? p.x + id * DK * p.dvp : p.init ? p.init + (int64_t)bh * p.dk_ * p.dv_ : nullptr;
  const Rsrc from_rs = make_rsrc(from);
  const unsigned from_ld = 4u * (ws ? p.dvp : p.dv_);
  const bool from_col = from && (ws ? value : in_v);
#pragma unroll
  for (int t = 0; t < ST; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 16 * t + 4 * g + i;
      if (MAP)
        S[t][i] = !value && row == col - p.dvp ? 1.0f : 0.0f;
      else
        S[t][i] = raw_value<float>(load_raw<float>(from_rs, from_col && (ws || row < p.dk_) ? row * from_ld + 4u * col : kOut));
    }
  const T* const kp = row_ptr<T>(p.k, b, 0, hk);
  const T* const qp = row_ptr<T>(p.q, b, 0, hk);
  const T* const vp = row_ptr<T>(p.v, b, 0, h);
  T* const op = MAP ? nullptr : row_ptr<T>(p.o, b, 0, h);
  const unsigned es = sizeof(T), v_row = (unsigned)p.v.ss * es, o_row = (unsigned)p.o.ss * es;
  const unsigned v_at = in_v ? col * es + 4 * g * v_row : kOut, o_at = in_v ? col * es + 4 * g * o_row : kOut;
  constexpr int NZ = (kZFloats / 4 + NT - 1) / NT;
  Block<T, KS, NT> kb, qb;
  f32x4 zr[NZ];
  unsigned vr[16];
  float gr[2];
  // The next chunk's inputs, each as soon as its registers are free (and left as
  // loaded: a conversion would wait for them here).
  auto rows_of = [&](int c) { return min(kDeltaChunk, tokens - c * kDeltaChunk); };
  auto fetch_k = [&](int c) { kb.load(kp + (int64_t)c * kDeltaChunk * p.k.ss, p.k.ss, rows_of(c), p.dk_, p.vec); };
  auto fetch_v = [&](int c) {
    const Rsrc rs = rows_rsrc<T>(vp + (int64_t)c * kDeltaChunk * p.v.ss, p.v.ss, rows_of(c), p.dv_);
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) vr[4 * t + i] = load_raw<T>(rs, v_at, (16 * t + i) * v_row);
  };
  auto fetch = [&](int c) {
    const int64_t chunk = (int64_t)bh * p.N + c;
    if (!MAP) qb.load(qp + (int64_t)c * kDeltaChunk * p.q.ss, p.q.ss, rows_of(c), p.dk_, p.vec);
#pragma unroll
    for (int e = 0; e < NZ; ++e) zr[e] = load4(p.z + chunk * kZFloats + 4 * min(tid + e * NT, kZFloats / 4 - 1));
#pragma unroll
    for (int e = 0; e < 2; ++e) gr[e] = p.gates[chunk * kGateFloats + min(tid + e * NT, kGateFloats - 1)];
  };
  auto put_gates = [&](int c) {
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (tid + e * NT < kGateFloats) gates[c & 1][tid + e * NT] = gr[e];
  };
  if (c0 < c1) {
    fetch_k(c0);
    fetch(c0);
    fetch_v(c0);
    put_gates(c0);
    // P's zeros beside the diagonal tiles that begin a pair
    if (!MAP)
      for (int e = tid; e < 32 * 3 * 4; e += NT) {
        const int row = (e & 31) < 16 ? (e & 31) : 16 + (e & 31), k = (e >> 5) % 3, q = 4 * (row >> 5 << 1) + 4 + (e >> 5) / 3;
        *reinterpret_cast<u32x2*>(&pp[MAP ? 0 : k][tri_at(row) + place4(q)]) = u32x2{0, 0};
      }
  }
  for (int c = c0; c < c1; ++c) {
    const int64_t t0 = (int64_t)c * kDeltaChunk;
    const float* const gt = gates[c & 1];
    __syncthreads();   // the chunk before has been read, this one's gates are there
    kb.template put_rows<LDK>(kk, kIn);
    if (MAP || kApart) kb.template put_columns<LKT>(kt, kIn);
    if (!MAP) qb.template put_rows<LDK>(qq, kIn);
    // -Z beta
#pragma unroll
    for (int e = 0; e < NZ; ++e) {
      const int quad = tid + e * NT;
      if (quad < kZFloats / 4) {
        u32x2 part[3];
        split4<3>(part, -zr[e] * load4(gt + kBeta + 4 * z_quad(quad)));
#pragma unroll
        for (int k = 0; k < 3; ++k) *reinterpret_cast<u32x2*>(&zp[k][tri_at(z_row(quad)) + place4(z_quad(quad))]) = part[k];
      }
    }
    __syncthreads();
    if (c + 1 < c1) {
      fetch(c + 1);
      if (MAP || kApart) fetch_k(c + 1);
    }
    if (!MAP) {
      // P, ten 16x16 tiles: four columns of one row a lane, from K Q^T
#pragma unroll
      for (int e = 0; e < (9 + WAVES) / WAVES; ++e) {
        const int tile = wave + WAVES * e;
        if (tile < 10) {
          const int tr = tile < 1 ? 0 : tile < 3 ? 1 : tile < 6 ? 2 : 3, tc = tile - tr * (tr + 1) / 2, i = 16 * tr + r;
          f32x4 acc = zero4();
          u32x4 kf[KS][NP], qf[KS][NP];
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            read_parts<NP>(kf[s], kk, kIn, (16 * tc + r) * LDK + 32 * s + 8 * g);
            read_parts<NP>(qf[s], qq, kIn, i * LDK + 32 * s + 8 * g);
          }
#pragma unroll
          for (int s = 0; s < KS; ++s) mul<NP, 2>(acc, kf[s], qf[s]);
          const f32x4 hi = load4(gt + kHi + 16 * tc + 4 * g), lo = load4(gt + kLo + 16 * tc + 4 * g);
          const float hi_i = gt[kHi + i], lo_i = gt[kLo + i];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            acc[k] = i >= 16 * tc + 4 * g + k ? acc[k] * __builtin_amdgcn_exp2f((hi_i - hi[k]) + (lo_i - lo[k])) : 0.0f;
          u32x2 part[3];
          split4<3>(part, acc);
#pragma unroll
          for (int k = 0; k < 3; ++k)
            *reinterpret_cast<u32x2*>(&pp[MAP ? 0 : k][tri_at(i) + 32 * (tc >> 1) + 8 * g + 4 * (tc & 1)]) = part[k];
        }
      }
    }
    f32x4 x[4], o[4];
    if (live) {
      if (!MAP && p.s && value) {
        float* const sg = p.s + ((int64_t)bh * p.N + c) * DK * p.dvp + col;
#pragma unroll
        for (int t = 0; t < ST; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) sg[(int64_t)(16 * t + 4 * g + i) * p.dvp] = S[t][i];
      }
      clear(x);
      clear(o);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        u32x4 sp[3];
        split_pair<3>(sp, S[2 * s], S[2 * s + 1]);
        products<NP, (NP == 1 ? 3 : 1), (MAP ? 4 : 8)>(
            kIn, [&](int i) { return (i < 4 ? kk : qq) + (16 * (i & 3) + r) * LDK + 32 * s + 8 * g; },
            [&](int i, const u32x4(&a)[NP]) {
              mul<3, 2>(i < 4 ? x[i & 3] : o[i & 3], a, sp);
            });
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const f32x4 gam = load4(gt + kGam + 16 * t + 4 * g);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[t][i] = raw_value<T>(vr[4 * t + i]) - gam[i] * x[t][i];
      }
    }
    if (c + 1 < c1) fetch_v(c + 1);
    if (!MAP) {
      __syncthreads();   // P is there, Q has been read
      if (!kApart) {
        kb.template put_columns<LKT>(kt, kIn);
        if (c + 1 < c1) fetch_k(c + 1);
      }
    }
    if (live) {
      // Y, on X's registers: the parts of X are taken first
      u32x4 xp[2][3];
      split_pair<3>(xp[0], x[0], x[1]);
      split_pair<3>(xp[1], x[2], x[3]);
      // tiles (t, s): (0, 0) .. (3, 0), (2, 1), (3, 1)
      products<3, 1, 6>(
          kTri, [&](int i) { return &zp[0][0] + tri_at(16 * (i < 4 ? i : i - 2) + r) + 32 * (i >> 2) + 8 * g; },
          [&](int i, const u32x4(&a)[3]) { mul<3, 2>(x[i < 4 ? i : i - 2], a, xp[i >> 2]); });
#pragma unroll
      for (int t = 0; t < 4; ++t) x[t] *= load4(gt + kBeta + 16 * t + 4 * g);   // U
      if (!MAP) {
#pragma unroll
        for (int t = 0; t < 4; ++t) o[t] *= load4(gt + kGam + 16 * t + 4 * g);
        u32x4 up[2][3];
        split_pair<3>(up[0], x[0], x[1]);
        split_pair<3>(up[1], x[2], x[3]);
        products<3, 1, 6>(
            kTri, [&](int i) { return &pp[0][0] + tri_at(16 * (i < 4 ? i : i - 2) + r) + 32 * (i >> 2) + 8 * g; },
            [&](int i, const u32x4(&a)[3]) { mul<3, 2>(o[i < 4 ? i : i - 2], a, up[i >> 2]); });
        const int rows = tokens - (int)t0;
        if (rows < kDeltaChunk)   // zeros past the tokens in use
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (16 * t + 4 * g + i >= rows) o[t][i] = 0.0f;
        const Rsrc o_rs = rows_rsrc<T>(op + t0 * p.o.ss, p.o.ss, min(kDeltaChunk, p.S - (int)t0), p.dv_);
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) store_one<T>(o_rs, o_at, (16 * t + i) * o_row, p.scale * o[t][i]);
      }
    }
    if (!MAP && !kApart) __syncthreads();   // K by columns is there
    if (live) {
      const float last = gt[kGam + 63];
#pragma unroll
      for (int t = 0; t < ST; ++t) S[t] *= last;
      u32x4 up[2][3];
#pragma unroll
      for (int s = 0; s < 2; ++s)
        split_pair<3>(up[s], x[2 * s] * load4(gt + kEnd + 32 * s + 4 * g), x[2 * s + 1] * load4(gt + kEnd + 32 * s + 16 + 4 * g));
      products<NP, (NP == 1 ? 3 : 1), 2 * ST>(
          kIn, [&](int i) { return kt + (16 * (i % ST) + r) * LKT + 32 * (i / ST) + 8 * g; },
          [&](int i, const u32x4(&a)[NP]) { mul<3, 2>(S[i % ST], a, up[i / ST]); });
    }
    if (c + 1 < c1) put_gates(c + 1);
  }
  if (MAP && live) {
    float* const dst = value ? p.x + id * DK * p.dvp + col : p.a + id * DK * DK + (col - p.dvp);
    const int ld = value ? p.dvp : DK;
#pragma unroll
    for (int t = 0; t < ST; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) dst[(int64_t)(16 * t + 4 * g + i) * ld] = S[t][i];
  }
  if (fin && in_v) {
    float* const dst = p.fin + (int64_t)bh * p.dk_ * p.dv_ + col;
#pragma unroll
    for (int t = 0; t < ST; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (16 * t + 4 * g + i < p.dk_) dst[(int64_t)(16 * t + 4 * g + i) * p.dv_] = S[t][i];
  }
}

template <typename T, int KS, bool MAP>
void launch_walk(const DeltaParams& p, hipStream_t stream) {
  const int slices = p.dvp / kDeltaSlice + (MAP ? p.dkp / kDeltaSlice : 0);
  auto go = [&](auto waves) {
    constexpr int W = decltype(waves)::value;
    const int groups = (slices + W - 1) / W;
    const unsigned grid = (unsigned)((int64_t)p.B * p.H * p.segs * groups);
    hipLaunchKernelGGL((delta_walk_kernel<T, KS, W, MAP>), dim3(grid), dim3(64 * W), 0, stream, p, groups);
  };
  // Eight waves share the first operands between more columns; four, where a CU
  // holds two such workgroups or more, wait less for each other.  Measured with four
  // and eight, B=1 S=8192 H=16: maps of bf16 dk=64 dv=128 148 and 165 us (the whole
  // forward), dk=dv=128 290 and 286, of fp32 dk=64 223 and 234, but dk=dv=128, one
  // workgroup a CU, 567 and 478; outputs of bf16 dk=64 dv=128 168 and 159, dk=dv=128
  // 387 and 296, of fp32 dk=64 285 and 234.  With dv=64 four waves hold every column:
  // bf16 dk=32 97 and 110, dk=64 121 and 136, but dk=96 194 and 178, dk=128 266 and 253;
  // fp32 dk=64 198 and 192, dk=128 408 and 454.
  constexpr bool kFour = MAP && (sizeof(T) == 2 || KS <= 2);
  if constexpr (kFour)
    go(std::integral_constant<int, 4>{});
  else if (slices <= 4)
    go(std::integral_constant<int, 4>{});
  else
    go(std::integral_constant<int, 8>{});
}

template <typename T, int KS>
hipError_t forward(const DeltaParams& p, hipStream_t stream) {
  const int64_t chunks = (int64_t)p.B * p.H * p.N;
  hipLaunchKernelGGL((delta_solve_kernel<T, KS>), dim3((unsigned)chunks), dim3(64), 0, stream, p);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && p.segs > 1) {
    launch_walk<T, KS, true>(p, stream);
    e = hipGetLastError();
    if (e == hipSuccess)
      e = launch_delta_scan(p, p.a, p.x, p.init, p.segs, p.seg * kDeltaChunk, false, stream);
  }
  if (e != hipSuccess) return e;
  launch_walk<T, KS, false>(p, stream);
  return hipGetLastError();
}

template <typename T>
hipError_t forward_by_size(const DeltaParams& p, hipStream_t stream) {
  switch (p.dkp / 32) {
    case 1: return forward<T, 1>(p, stream);
    case 2: return forward<T, 2>(p, stream);
    case 3: return forward<T, 3>(p, stream);
    default: return forward<T, 4>(p, stream);
  }
}

}  // namespace

// Chunks a segment.  A segmented row is walked twice, on top of a scan, but by many
// workgroups: worth it for up to 128 heads (bf16, d = 64, whole rows against
// segments: 128 heads x 64 chunks 382 and 303 us, 160 x 51 317 and 376, 192 x 42 273
// and 324; 16 x 512 2609 and 335) and from 4 chunks (8 heads x 4 34.8 and 31.3 us,
// x 8 54.8 and 35.7).  At most as many segments as give every CU two workgroups: one
// more and a third round of them begins (96 heads x 85 chunks: 5 segments 306 us, 6
// 366).  Below that a walk costs its segment's length and the scan their number, so
// the best length goes with the root of the row's: with 1, 2, 3, 4 chunks a segment
// 8 heads x 16 chunks take 43.9, 44.6, 49.1, 55.3 us, x 47 76.5, 62.7, 60.2, 64.8,
// x 128 165, 113, 99, 90 (8: 101); fp32 and d = 128 have theirs at the same lengths.
int delta_segment(int64_t heads, int64_t chunks) {
  if (heads > 128 || chunks < 4) return (int)std::max<int64_t>(chunks, 1);
  const int64_t most = 512 / std::max<int64_t>(heads, 1);
  return (int)std::max<int64_t>((chunks + most - 1) / most, (int64_t)(std::sqrt(chunks / 6.0) + 0.5));
}

hipError_t launch_delta_scan(const DeltaParams& p, const float* a, float* x, const float* init, int n, int span,
                             bool reverse, hipStream_t stream) {
  const int BH = p.B * p.H, ns = p.dvp / kDeltaSlice;
  const dim3 grid((unsigned)(8 * (int64_t)ns * ((BH + 7) / 8)));
  auto go = [&](auto kt) {
    constexpr int KT = decltype(kt)::value;
    hipLaunchKernelGGL((delta_scan_kernel<KT>), grid, dim3(64 * KT), 0, stream, a, x, init, p.lengths, p.S, n, span,
                       BH, p.H, p.dk_, p.dv_, p.dvp, reverse);
  };
  switch (p.dkp / 32) {
    case 1: go(std::integral_constant<int, 2>{}); break;
    case 2: go(std::integral_constant<int, 4>{}); break;
    case 3: go(std::integral_constant<int, 6>{}); break;
    default: go(std::integral_constant<int, 8>{}); break;
  }
  return hipGetLastError();
}

hipError_t launch_delta_fwd(const DeltaParams& p, int dtype, hipStream_t stream) {
  return dtype == 0 ? forward_by_size<float>(p, stream) : forward_by_size<__bf16>(p, stream);
}

}  // namespace osm
