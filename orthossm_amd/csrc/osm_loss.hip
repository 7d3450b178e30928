// The cross entropy of a projection to a vocabulary on gfx950, without its logits.
//
//   l = W h,  lse = log sum_v e^{l_v},  loss = lse - l_target
//   P = (e^{l - lse} - [v = target]) g,   dH = P W,   dW = P^T H
//
// Forward: a workgroup forms a tile of logits by classes and tokens in its
// accumulators and leaves of it, for every token, the largest and the sum of
// exponentials below it (an online softmax over tiles); a second kernel joins the tiles.  Backward, a piece of the
// vocabulary at a time: the logits again, from them P (to bf16, of few tokens to two bf16
// parts, of fp32 to three), then the two products, which read W, P and H by columns where they
// have to.  What counts for all of them: the products' operations on the matrix
// instruction (osm_gemm.h); the tokens that do not count are left out first, so they
// cost nothing.  Exponentials and logarithms are those of 2: l log2(e) less the largest
// is one fused operation, and what its rounding leaves out cancels in the loss.
//
// 8192 tokens, 50001 classes, 1024 columns, bf16: forward 813 to 900 us from GPU to GPU (1030 to
// 930 TFLOP/s; the product alone 680; its epilogue, which nothing overlaps, takes 12%, most of it
// the exponentials), P 930, dH 850, dW 820; a library's product for the logits alone takes 815,
// with 0.8 GB of them written.  4096 tokens, 32768 classes, 1024 columns, forward: 255 us,
// 1080 TFLOP/s.  981 tokens of 1401, 5003 classes, 400 columns, fp32: 39, 43, 37, 46 us, of 6
// products of 4 GFLOP each.
#include <algorithm>
#include <type_traits>

#include "osm_gemm.h"
#include "osm_loss.h"
#include "osm_wide_store.h"

namespace osm {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504f, kLn2 = 0.693147181f, kInf = __builtin_inff();

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// ---- operands ----

constexpr float kMostBf16 = 0x1.fep127f;

// The bf16 parts of x: part k is what rounding leaves of the parts before it.  (The first of
// what bf16 would round to infinity is its largest; of an infinity it is one, and the others are
// of no use.)
template <int PARTS>
__device__ __forceinline__ void split(float x, __bf16 (&to)[PARTS]) {
#pragma unroll
  for (int k = 0; k < PARTS; ++k) {
    const bool clamp = PARTS > 1 && k == 0 && __builtin_fabsf(x) < kInf;
    to[k] = (__bf16)(clamp ? __builtin_fmaxf(__builtin_fminf(x, kMostBf16), -kMostBf16) : x);
    x -= (float)to[k];
  }
}

// 8 columns from c on of a row of D, zeros past them, as parts.
template <typename T, int PARTS>
__device__ __forceinline__ void split_unit(const T* row, int c, int D, bool vec, bf16x8 (&out)[PARTS]) {
  typedef T V8 __attribute__((ext_vector_type(8)));
  V8 v = {};
  if (vec) {   // (rows of whole units at multiples of 16 bytes)
    if (c < D) v = *reinterpret_cast<const V8*>(row + c);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (c + k < D) v[k] = row[c + k];
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    __bf16 s[PARTS];
    split<PARTS>((float)v[k], s);
#pragma unroll
    for (int q = 0; q < PARTS; ++q) out[q][k] = s[q];
  }
}

template <typename T>
bool whole_units(const void* p, int64_t stride, int64_t D) {
  return (uintptr_t)p % 16 == 0 && stride * sizeof(T) % 16 == 0 && D % 8 == 0;
}

// A piece's rows of weights to [PARTS][vn][Dpad].
template <typename T, int PARTS>
__device__ __forceinline__ void pack(const LossParams& p, __bf16* to, bool vec, int64_t block) {
  const int units = p.Dpad / 8;
  const int64_t i = block * 256 + threadIdx.x, n = p.vn;
  if (i >= n * units) return;
  const int64_t r = i / units;
  const int c = (int)(i - r * units) * 8;
  bf16x8 out[PARTS];
  split_unit<T, PARTS>(static_cast<const T*>(p.weight) + (p.v0 + r) * p.weight_s, c, (int)p.D, vec, out);
#pragma unroll
  for (int q = 0; q < PARTS; ++q) {
    *reinterpret_cast<bf16x8*>(to + (q * n + r) * p.Dpad + c) = out[q];
    wide_store_wait();
  }
}
template <typename T, int PARTS>
__global__ void __launch_bounds__(256) loss_pack_kernel(const LossParams p, __bf16* to, bool vec) {
  pack<T, PARTS>(p, to, vec, blockIdx.x);
}

// The tokens that count, one after the other: a block takes `each` tokens, counts those
// before them, and writes where its own go, and their hidden rows.  The blocks after those take
// the first piece's weights (981 tokens, 5003 classes, 400 columns, fp32: 10 us for
// 7 and 6, and a launch less twice a step, 180 us for 196).
template <typename T, int PARTS>
__global__ void __launch_bounds__(256) loss_rows_kernel(const LossParams p, __bf16* to, int64_t each, int blocks, bool vec, __bf16* w,
                                                          bool w_vec, bool bwd) {
  if ((int)blockIdx.x >= blocks) {
    pack<T, PARTS>(p, w, w_vec, (int)blockIdx.x - blocks);
    return;
  }
  __shared__ int sums[4];
  __shared__ int rows[256];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  auto in_order = [&](bool in, int& base) {   // this thread's place from `base` on; base: after all of them
    const unsigned long long mask = __ballot(in);
    __syncthreads();
    if (lane == 0) sums[wave] = __popcll(mask);
    __syncthreads();
    int at = base + __popcll(mask & ((1ull << lane) - 1));
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (w < wave) at += sums[w];
      base += sums[w];
    }
    return at;
  };
  const int64_t t0 = blockIdx.x * each, t1 = min(t0 + each, p.N);
  int before = 0;
  for (int64_t i = threadIdx.x; i < t0; i += 256) before += p.targets[i] != p.ignore;
#pragma unroll
  for (int w = 32; w > 0; w >>= 1) before += __shfl_xor(before, w);
  if (lane == 0) sums[wave] = before;
  __syncthreads();
  int base = sums[0] + sums[1] + sums[2] + sums[3];
  const int units = p.Dpad / 8;
  for (int64_t i0 = t0; i0 < t1; i0 += 256) {
    const int64_t i = i0 + threadIdx.x;
    const bool in = i < t1 && p.targets[i] != p.ignore;
    const int first = base, at = in_order(in, base);
    if (in) {
      const int64_t target = p.targets[i];
      p.tok.targets[at] = target >= 0 && target < p.V ? (int)target : -1;
      if (bwd) p.tok.factors[at] = make_float2(p.lse[i] * kLog2e, p.grad_losses ? p.grad_losses[i] : 1.0f);
      rows[at - first] = (int)i;
    }
    if (i < t1) p.tok.places[i] = in ? at : -1;
    __syncthreads();
    const int n = (base - first) * units;
    constexpr int kAtOnce = 4;   // (loads on their way)
    for (int u0 = threadIdx.x; u0 < n; u0 += 256 * kAtOnce) {
      bf16x8 out[kAtOnce][PARTS];
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        const int u = min(u0 + 256 * k, n - 1), r = u / units;
        split_unit<T, PARTS>(static_cast<const T*>(p.hidden) + rows[r] * p.hidden_s, 8 * (u - r * units), (int)p.D, vec, out[k]);
      }
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        const int u = u0 + 256 * k;
#pragma unroll
        for (int q = 0; q < PARTS; ++q)
          if (u < n) {
            *reinterpret_cast<bf16x8*>(to + ((int64_t)q * p.Npad + first) * p.Dpad + 8 * (int64_t)u) = out[k][q];
            wide_store_wait();
          }
      }
    }
  }
  if ((int)blockIdx.x < blocks - 1) return;
  if (threadIdx.x == 0) *p.tok.count = base;
  // zeros up to a whole step of the products over tokens
  const int over = (base + kStep - 1) / kStep * kStep - base;
  for (int u = threadIdx.x; u < PARTS * over * units; u += 256) {
    const int q = u / (over * units), r = u - q * over * units;
    *reinterpret_cast<bf16x8*>(to + ((int64_t)q * p.Npad + base) * p.Dpad + 8 * (int64_t)r) = bf16x8{};
    wide_store_wait();
  }
}

// ---- products ----

// A block's tile (m, n) of tm by tn: the XCDs, to which blocks go in turn, take
// contiguous shares of an order that walks bands of 8 columns by rows, so that what is
// at work on an XCD at a time shares rows and columns in its L2.  False: no tile.
__device__ __forceinline__ bool tile_of(int tm, int tn, int& m, int& n) {
  const int total = tm * tn, share = (total + 7) / 8, id = (blockIdx.x & 7) * share + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= share || id >= total) return false;
  const int band = id / (8 * tm), rest = id - band * 8 * tm, width = min(8, tn - band * 8);
  m = rest / width;
  n = band * 8 + rest - m * width;
  return true;
}
// Tiles of the tokens that count, over which the XCDs are shared out: over all tokens', some XCDs
// would have none to form, and the others as many as ever (4096 tokens, 32768 classes of 1024,
// 278 us: with 30% of them left out the same, and 210).
template <class G>
__device__ __forceinline__ int tiles_of(int count) {
  return (count + G::TN - 1) / G::TN;
}
unsigned grid_of(int64_t tm, int64_t tn) { return (unsigned)((tm * tn + 7) / 8 * 8); }

GemmSide side(const __bf16* p, int64_t ld, int64_t part, int rows, int cols) { return {p, ld, part, rows, cols}; }

struct Product {
  GemmSide a, b;
  int tm, tn;
};

// Logits of a tile: A the piece's classes, B the tokens that count.  BWD false: the
// tile's largest logit and sum of exponentials for each token, and the target's logit.
// BWD true: P.
template <class G, bool BWD>
__global__ void __launch_bounds__(G::kThreads) loss_logits_kernel(const LossParams p, const Product g) {
  __shared__ __attribute__((aligned(16))) __bf16 lds[G::kLds];
  const bool all = !BWD && !p.tok.count;
  const int count = all ? (int)p.N : *p.tok.count;
  int tm, tn;
  if (!tile_of(g.tm, tiles_of<G>(count), tm, tn)) return;
  const int m0 = tm * G::TM, n0 = tn * G::TN;
  const GemmPlace<G> q;
  const int rows = p.vn - m0;   // of the tile that are classes
  // Of column j's token: its target as a row of the tile, -1 if it is none that this wave
  // holds, and its factors.  (Read here: after the product nothing would hide the way.)
  int aim[G::FN];
  float2 factors[G::FN];
#pragma unroll
  for (int j = 0; j < G::FN; ++j) {
    const int n = min(n0 + q.col(j), count - 1);
    int64_t t = all ? p.targets[n] : p.tok.targets[n];
    t = t < p.V ? t - p.v0 - m0 : -1;
    aim[j] = n0 + q.col(j) < count && t >= q.m && t < min(q.m + G::TM / G::WM, rows) ? (int)t : -1;
    if (BWD) factors[j] = p.tok.factors[n];
  }
  f32x16 acc[G::FM][G::FN];
  zero<G>(acc);
  gemm<G, false, false>(g.a, g.b, m0, n0, 0, p.Dpad / kStep, lds, acc);
  // f(value, row) for the rows that a lane holds of column j; change: what it gives takes the value's place
  auto each = [&](int j, auto f) {
#pragma unroll
    for (int s = 0; s < G::FM; ++s)
#pragma unroll
      for (int i = 0; i < 16; ++i) f(acc[s][j][i], q.row(s, i));
  };
  auto change = [&](int j, auto f) {
#pragma unroll
    for (int s = 0; s < G::FM; ++s)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[s][j][i] = f(acc[s][j][i], q.row(s, i));
  };
  if constexpr (!BWD) {
    float2* const red = reinterpret_cast<float2*>(lds);   // [WM][TN]
#pragma unroll
    for (int j = 0; j < G::FN; ++j) {
      if (rows < G::TM) change(j, [&](float l, int m) { return m < rows ? l : -kInf; });
      if (__any(aim[j] >= 0)) each(j, [&](float l, int m) { if (m == aim[j]) p.own[n0 + q.col(j)] = l; });
      float top = -kInf, sum = 0.0f;
      each(j, [&](float l, int) { top = __builtin_fmaxf(top, l); });
      top = __builtin_fmaxf(top, __shfl_xor(top, 32)) * kLog2e;   // (the other half's rows)
      const float base = top == -kInf ? 0.0f : top;
      each(j, [&](float l, int) { sum += exp2_of(__builtin_fmaf(l, kLog2e, -base)); });
      sum += __shfl_xor(sum, 32);
      if (q.lane < 32) red[q.m / (G::TM / G::WM) * G::TN + q.col(j)] = make_float2(top, sum);
    }
    __syncthreads();
    for (int c = threadIdx.x; c < G::TN; c += G::kThreads) {
      float top = -kInf, sum = 0.0f;
#pragma unroll
      for (int w = 0; w < G::WM; ++w) top = __builtin_fmaxf(top, red[w * G::TN + c].x);
      const float b = top == -kInf ? 0.0f : top;
#pragma unroll
      for (int w = 0; w < G::WM; ++w) sum += red[w * G::TN + c].y * exp2_of(red[w * G::TN + c].x - b);
      p.stat[(int64_t)(p.tile0 + tm) * p.Npad + n0 + c] = make_float2(top, sum);
    }
  } else {
#pragma unroll
    for (int j = 0; j < G::FN; ++j) {
      const int n = n0 + q.col(j);
      change(j, [&](float l, int) { return exp2_of(__builtin_fmaf(l, kLog2e, -factors[j].x)); });
      if (__any(aim[j] >= 0)) change(j, [&](float e, int m) { return m == aim[j] ? e - 1.0f : e; });
      if (p.grad_losses) change(j, [&](float e, int) { return e * factors[j].y; });
      if (rows < G::TM || n0 + G::TN > count) change(j, [&](float e, int m) { return n < count && m < rows ? e : 0.0f; });
    }
    constexpr int kRowUnits = G::TM / 8;
    const int parts = G::PARTS > 1 ? G::PARTS : G::kFew ? p.p_parts : 1;
    static_assert(G::TM * G::TN <= G::kLds, "a tile of P fits");
#pragma unroll 1
    for (int part = 0; part < parts; ++part) {
      // a lane's four neighbouring classes are half a 16-byte unit, which lies at its index
      // xor its token's; then the next part is what rounding left
#pragma unroll
      for (int j = 0; j < G::FN; ++j)
#pragma unroll
        for (int f = 0; f < G::FM; ++f)
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            const int c = q.col(j), r = q.row(f, i);
            bf16x4 v;
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = (__bf16)acc[f][j][i + k];
            *reinterpret_cast<bf16x4*>(lds + c * G::TM + ((r / 8) ^ (c % kRowUnits)) * 8 + r % 8) = v;
          }
      __syncthreads();
      constexpr int kEach = G::TN * kRowUnits / G::kThreads, kAtOnce = kEach < 4 ? kEach : 4;   // units of a thread
      static_assert(G::kThreads % kRowUnits == 0 && kEach % kAtOnce == 0, "a thread's units are of one class");
      const int c0 = threadIdx.x / kRowUnits, r = threadIdx.x % kRowUnits;
      if (m0 + r * 8 < p.vpad) {
        __bf16* const to = p.p + ((int64_t)part * p.Npad + n0 + c0) * p.vpad + m0 + r * 8;
#pragma unroll
        for (int k = 0; k < kEach; k += kAtOnce) {
          bf16x8 v[kAtOnce];
#pragma unroll
          for (int i = 0; i < kAtOnce; ++i) {
            const int c = c0 + (k + i) * (G::kThreads / kRowUnits);
            v[i] = *reinterpret_cast<const bf16x8*>(lds + c * G::TM + (r ^ (c % kRowUnits)) * 8);
          }
#pragma unroll
          for (int i = 0; i < kAtOnce; ++i) {
            *reinterpret_cast<bf16x8*>(to + (int64_t)(k + i) * (G::kThreads / kRowUnits) * p.vpad) = v[i];
            wide_store_wait();
          }
        }
      }
      if (part + 1 == parts) break;
#pragma unroll
      for (int j = 0; j < G::FN; ++j) change(j, [&](float e, int) { return e - (float)(__bf16)e; });
      __syncthreads();
    }
  }
}

// f of P, whose parts a product of three part operands takes by itself; where few tokens'
// has two, each is a walk of its own.
template <class G, typename F>
__device__ __forceinline__ void over_parts(const LossParams& p, GemmSide b, F f) {
  const int n = G::kFew ? p.p_parts : 1;
#pragma unroll 1
  for (int i = 0; i < n; ++i, b.p += b.part) f(b);
}

// dH of a piece: A the weights by columns, B P; a split takes a share of the classes and
// adds to sums of its own.
template <class G>
__global__ void __launch_bounds__(G::kThreads) loss_dh_kernel(const LossParams p, const Product g) {
  __shared__ __attribute__((aligned(16))) __bf16 lds[G::kLds];
  const int across = tiles_of<G>(*p.tok.count);
  int tm, tn;
  if (!tile_of(g.tm, across * p.splits, tm, tn)) return;   // (a split beside the other: an XCD's tiles are of few of them)
  const int split = tn / across, m0 = tm * G::TM, n0 = (tn - split * across) * G::TN;
  const int all = p.vpad / kStep, each = (all + p.splits - 1) / p.splits, s0 = min(split * each, all);
  f32x16 acc[G::FM][G::FN];
  zero<G>(acc);
  over_parts<G>(p, g.b, [&](const GemmSide& b) {
    gemm<G, true, false>(g.a, b, m0, n0, (int64_t)s0 * kStep, min(each, all - s0), lds, acc);
  });
  const GemmPlace<G> q;
#pragma unroll
  for (int j = 0; j < G::FN; ++j) {
    float* const to = p.dh + ((int64_t)split * p.Npad + n0 + q.col(j)) * p.Dpad;
#pragma unroll
    for (int f = 0; f < G::FM; ++f)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int m = m0 + q.row(f, i);
        if (m >= p.Dpad) continue;
        f32x4 v = {acc[f][j][i], acc[f][j][i + 1], acc[f][j][i + 2], acc[f][j][i + 3]};
        if (!p.first) v += *reinterpret_cast<const f32x4*>(to + m);
        *reinterpret_cast<f32x4*>(to + m) = v;
        wide_store_wait();
      }
  }
}

__device__ __forceinline__ float factor(const LossParams& p) {
  return (p.grad ? *p.grad : 1.0f) / (p.count_in ? *p.count_in : 1.0f);
}

// dW of a piece: A the hidden rows, B P, both by columns.
template <class G, typename T>
__global__ void __launch_bounds__(G::kThreads) loss_dw_kernel(const LossParams p, const Product g) {
  __shared__ __attribute__((aligned(16))) __bf16 lds[G::kLds];
  int tm, tn;
  if (!tile_of(g.tm, g.tn, tm, tn)) return;
  const int m0 = tm * G::TM, n0 = tn * G::TN;
  f32x16 acc[G::FM][G::FN];
  zero<G>(acc);
  over_parts<G>(p, g.b, [&](const GemmSide& b) {
    gemm<G, true, true>(g.a, b, m0, n0, 0, (*p.tok.count + kStep - 1) / kStep, lds, acc);
  });
  const float s = factor(p);
  const GemmPlace<G> q;
  typedef T V4 __attribute__((ext_vector_type(4)));
  const bool vec = p.D % 4 == 0;
#pragma unroll
  for (int j = 0; j < G::FN; ++j) {
    const int n = n0 + q.col(j);
    if (n >= p.vn) continue;
    T* const to = static_cast<T*>(p.grad_w) + (p.v0 + n) * p.D;
#pragma unroll
    for (int f = 0; f < G::FM; ++f)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int m = m0 + q.row(f, i);
        V4 v;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = (T)(acc[f][j][i + k] * s);
        if (vec) {
          if (m < p.D) {
            *reinterpret_cast<V4*>(to + m) = v;
            if (sizeof(V4) > 8) wide_store_wait();
          }
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (m + k < p.D) to[m + k] = v[k];
        }
      }
  }
}

// ---- joins ----

constexpr int kJoinTokens = 16, kJoinSlices = 16;

// The sum of d over a workgroup of T threads in its first, in an order that does not depend
// on timing.
template <int T>
__device__ __forceinline__ double block_sum(double d, double* red) {
  red[threadIdx.x] = d;
  for (int w = T / 2; w > 0; w >>= 1) {
    __syncthreads();
    if ((int)threadIdx.x < w) red[threadIdx.x] += red[threadIdx.x + w];
  }
  return red[0];
}

// A token's statistics over the vocabulary's tiles, 16 threads a token; zeros of those
// that do not count.
__global__ void __launch_bounds__(kJoinTokens * kJoinSlices) loss_join_kernel(const LossParams p, int tiles) {
  __shared__ float2 red[kJoinSlices][kJoinTokens];
  const int c = threadIdx.x % kJoinTokens, s = threadIdx.x / kJoinTokens;
  const int64_t token = (int64_t)blockIdx.x * kJoinTokens + c;
  int at = -1;
  if (token < p.N) at = p.tok.places ? p.tok.places[token] : p.targets[token] != p.ignore ? (int)token : -1;
  float top = -kInf, sum = 0.0f;
  if (at >= 0) {
#pragma unroll 4
    for (int t = s; t < tiles; t += kJoinSlices) {
      const float2 v = p.stat[(int64_t)t * p.Npad + at];
      const float both = __builtin_fmaxf(top, v.x), b = both == -kInf ? 0.0f : both;
      sum = sum * exp2_of(top - b) + v.y * exp2_of(v.x - b);
      top = both;
    }
  }
  red[s][c] = make_float2(top, sum);
  __syncthreads();
  if (s > 0 || token >= p.N) return;
  float loss = 0.0f, lse = 0.0f;
  if (at >= 0) {
    for (int k = 1; k < kJoinSlices; ++k) top = __builtin_fmaxf(top, red[k][c].x);
    const float b = top == -kInf ? 0.0f : top;
    sum = 0.0f;
    for (int k = 0; k < kJoinSlices; ++k) sum += red[k][c].y * exp2_of(red[k][c].x - b);
    const int64_t target = p.targets[token];
    const bool known = target >= 0 && target < p.V;
    const float l = log2f(sum);
    lse = known ? (b + l) * kLn2 : __builtin_nanf("");
    // (small losses keep their digits)
    loss = known ? (l - __builtin_fmaf(p.own[at], kLog2e, -b)) * kLn2 : __builtin_nanf("");
  }
  p.lse[token] = lse;
  if (p.losses) p.losses[token] = loss;
}

// The sum of the losses in double, one workgroup, in an order that does not depend on timing.
__global__ void __launch_bounds__(1024) loss_total_kernel(const LossParams p) {
  __shared__ double red[1024], counts[1024];
  double s = 0.0, n = 0.0;
  for (int64_t i = threadIdx.x; i < p.N; i += 1024) {
    s += p.losses[i];
    if (!p.tok.count) n += p.targets[i] != p.ignore;
  }
  s = block_sum<1024>(s, red);
  n = p.tok.count ? *p.tok.count : block_sum<1024>(n, counts);
  if (threadIdx.x == 0) {
    n = n < 1.0 ? 1.0 : n;
    *p.loss = (float)(p.mean ? s / n : s);
    if (p.count) *p.count = (float)n;
  }
}

// The loss of no tokens.
__global__ void loss_none_kernel(float* loss, float* count) {
  if (loss) *loss = 0.0f;
  if (count) *count = 1.0f;
}

// grad_h of every token from its place's sums, zeros where it does not count.
template <typename T>
__global__ void __launch_bounds__(256) loss_finish_kernel(const LossParams p) {
  const int64_t per = (p.D + 3) / 4, all = p.N * per;
  const float s = factor(p);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int64_t n = i / per;
    const int d = (int)(i - n * per) * 4, at = p.tok.places[n];
    f32x4 v = {};
    if (at >= 0) {
      for (int k = 0; k < p.splits; ++k) v += *reinterpret_cast<const f32x4*>(p.dh + ((int64_t)k * p.Npad + at) * p.Dpad + d);
      v *= s;
    }
    T* const to = static_cast<T*>(p.grad_h) + n * p.D + d;
    typedef T V4 __attribute__((ext_vector_type(4)));
    V4 o;
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = (T)v[k];
    if (p.D % 4 == 0) {
      *reinterpret_cast<V4*>(to) = o;
      if (sizeof(V4) > 8) wide_store_wait();
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (d + k < p.D) to[k] = o[k];
    }
  }
}

// Zeros of a gradient that no token has a part in.
template <typename T>
__global__ void __launch_bounds__(256) loss_zero_kernel(T* to, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) to[i] = (T)0.0f;
}

constexpr int kCUs = 256;

// The largest tile of which the CUs get as many as they hold, or nearly, else the next; none
// that is more than twice as wide as the product.  Measured in us, the larger and the smaller:
//   50176 classes x 8192 tokens x 1024, the first and the second: 680, 855
//   64 tokens over 50001 classes of 1024, forward, the first and the third: 40, 27
//   1000 x 64 x 256, 8 of the third or 16 of the least: 4.0, 3.3
//   1024 x 849 x 8192, 56 of the second, 112 of the third, 224 of the least: 81, 71, 61
// (The least, alone on its CU, has two steps on their way: 43 for those 61, and 54 for 94 where
// rows lie 35 KB apart.  The others gain nothing by it, or lose a workgroup's room.)
// Three parts, the three tiles:
//   16384 x 4096 x 1024: 703, 791, 922
//   5003 x 981 x 448, 320, 640 and 1264 tiles: 38, 36, 37
//   448 x 5003 x 1024, 160, 316 and 553 tiles: 50, 47, 44
// The gradient of few tokens' weights has no use for the first tile, which could not hold what
// P's two parts take: it writes more than it multiplies.
template <typename F>
void by_size(const LossParams& p, int64_t M, int64_t N, F f) {
  auto tiles = [&](int64_t tm, int64_t tn) { return (M + tm - 1) / tm * ((N + tn - 1) / tn); };
  const int64_t least = std::min(M, N);
  if (p.parts == 1) {
    if (tiles(256, 256) >= kCUs * 3 / 4 && least > 128 && p.p_parts == 1)
      f(GemmTile<256, 256, 4, 2>{});
    else if (tiles(128, 128) >= kCUs * 3 / 2 && least > 64)
      f(GemmTile<128, 128, 2, 2>{});
    else if (tiles(128, 64) >= kCUs / 2)
      f(GemmTile<128, 64, 2, 2>{});
    else
      f(GemmTile<64, 64, 2, 2, 1, 3>{});
  } else {
    if (tiles(128, 128) >= kCUs * 3 && least > 64)
      f(GemmTile<128, 128, 4, 2, 3>{});
    else if (tiles(128, 64) >= kCUs * 2)
      f(GemmTile<128, 64, 2, 2, 3>{});
    else
      f(GemmTile<64, 64, 2, 2, 3>{});
  }
}

template <class G>
Product product(GemmSide a, GemmSide b, int64_t M, int64_t N) {
  return {a, b, (int)((M + G::TM - 1) / G::TM), (int)((N + G::TN - 1) / G::TN)};
}

template <bool BWD>
hipError_t logits(const LossParams& p, hipStream_t stream) {
  by_size(p, BWD ? p.vpad : p.V, p.N, [&](auto g) {
    using G = decltype(g);
    const Product t = product<G>(side(p.w, p.w_ld, p.w_part, p.vn, 0), side(p.h, p.h_ld, p.h_part, p.h_rows, 0),
                                 BWD ? p.vpad : p.vn, p.N);
    hipLaunchKernelGGL((loss_logits_kernel<G, BWD>), dim3(grid_of(t.tm, t.tn)), dim3(G::kThreads), 0, stream, p, t);
  });
  return hipGetLastError();
}

}  // namespace

namespace {
int64_t pack_blocks(const LossParams& p) { return ((int64_t)p.vn * (p.Dpad / 8) + 255) / 256; }

template <typename T, int PARTS>
void rows(const LossParams& p, __bf16* h, __bf16* w, bool bwd, hipStream_t stream) {
  // (a block counts what is before its tokens, so that there are at most 1024 of them)
  const int64_t each = std::max<int64_t>(4, (p.N + 1023) / 1024), blocks = (p.N + each - 1) / each;
  hipLaunchKernelGGL((loss_rows_kernel<T, PARTS>), dim3((unsigned)(blocks + (w ? pack_blocks(p) : 0))), dim3(256), 0, stream, p, h, each,
                     (int)blocks, whole_units<T>(p.hidden, p.hidden_s, p.D), w, whole_units<T>(p.weight, p.weight_s, p.D), bwd);
}
}  // namespace

hipError_t launch_loss_rows(const LossParams& p, __bf16* h, __bf16* w, int dtype, bool bwd, hipStream_t stream) {
  if (dtype == 0)
    rows<float, 3>(p, h, w, bwd, stream);
  else
    rows<__bf16, 1>(p, h, w, bwd, stream);
  return hipGetLastError();
}

hipError_t launch_loss_weight(const LossParams& p, __bf16* to, int dtype, hipStream_t stream) {
  const dim3 grid((unsigned)pack_blocks(p));
  if (dtype == 0)
    hipLaunchKernelGGL((loss_pack_kernel<float, 3>), grid, dim3(256), 0, stream, p, to, whole_units<float>(p.weight, p.weight_s, p.D));
  else
    hipLaunchKernelGGL((loss_pack_kernel<__bf16, 1>), grid, dim3(256), 0, stream, p, to, whole_units<__bf16>(p.weight, p.weight_s, p.D));
  return hipGetLastError();
}

int loss_tile_rows(const LossParams& p) {
  int rows = 0;
  by_size(p, p.V, p.N, [&](auto g) { rows = decltype(g)::TM; });
  return rows;
}

hipError_t launch_loss_logits(const LossParams& p, hipStream_t stream) { return logits<false>(p, stream); }
hipError_t launch_loss_probs(const LossParams& p, hipStream_t stream) { return logits<true>(p, stream); }

hipError_t launch_loss_join(const LossParams& p, int tiles, hipStream_t stream) {
  hipLaunchKernelGGL(loss_join_kernel, dim3((unsigned)((p.N + kJoinTokens - 1) / kJoinTokens)), dim3(kJoinTokens * kJoinSlices), 0, stream,
                     p, tiles);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !p.loss) return e;
  hipLaunchKernelGGL(loss_total_kernel, dim3(1), dim3(1024), 0, stream, p);
  return hipGetLastError();
}

hipError_t launch_loss_none(float* loss, float* count, hipStream_t stream) {
  hipLaunchKernelGGL(loss_none_kernel, dim3(1), dim3(1), 0, stream, loss, count);
  return hipGetLastError();
}

hipError_t launch_loss_dh(const LossParams& p, hipStream_t stream) {
  by_size(p, (int64_t)p.Dpad * p.splits, p.N, [&](auto g) {
    using G = decltype(g);
    const Product t = product<G>(side(p.w, p.w_ld, p.w_part, p.vn, p.Dpad), side(p.p, p.vpad, (int64_t)p.Npad * p.vpad, p.Npad, 0),
                                 p.D, p.N);
    hipLaunchKernelGGL((loss_dh_kernel<G>), dim3(grid_of(t.tm, t.tn * p.splits)), dim3(G::kThreads), 0, stream, p, t);
  });
  return hipGetLastError();
}

hipError_t launch_loss_dw(LossParams p, int from, int n, hipStream_t stream) {
  p.v0 += from;
  p.vn = n;
  by_size(p, p.D, n, [&](auto g) {
    using G = decltype(g);
    using T = std::conditional_t<G::PARTS == 1, __bf16, float>;
    const Product t = product<G>(side(p.h, p.h_ld, p.h_part, p.h_rows, p.Dpad),
                                 side(p.p + from, p.vpad, (int64_t)p.Npad * p.vpad, p.Npad, p.vpad - from), p.D, n);
    hipLaunchKernelGGL((loss_dw_kernel<G, T>), dim3(grid_of(t.tm, t.tn)), dim3(G::kThreads), 0, stream, p, t);
  });
  return hipGetLastError();
}

hipError_t launch_loss_zero(void* to, int64_t n, int dtype, hipStream_t stream) {
  const dim3 grid((unsigned)std::min<int64_t>((n + 255) / 256, 4096));
  if (dtype == 0)
    hipLaunchKernelGGL((loss_zero_kernel<float>), grid, dim3(256), 0, stream, static_cast<float*>(to), n);
  else
    hipLaunchKernelGGL((loss_zero_kernel<__bf16>), grid, dim3(256), 0, stream, static_cast<__bf16*>(to), n);
  return hipGetLastError();
}

hipError_t launch_loss_finish(const LossParams& p, int dtype, hipStream_t stream) {
  const dim3 grid((unsigned)std::min<int64_t>((p.N * ((p.D + 3) / 4) + 255) / 256, 1 << 16));
  if (dtype == 0)
    hipLaunchKernelGGL((loss_finish_kernel<float>), grid, dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((loss_finish_kernel<__bf16>), grid, dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace osm
