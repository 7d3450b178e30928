// Parameters of the gated delta rule's kernels (osm_delta.hip,
// osm_delta_bwd.hip) and the tile products both are built from.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace osm {

constexpr int kDeltaChunk = 64;      // tokens a chunk
constexpr int kDeltaMaxDk = 128;     // rows of the state
constexpr int kDeltaSlice = 16;      // columns of the state a scan workgroup holds

// Rows of a token tensor: element (b, t, h, j) at b*sb + t*ss + h*sh + j.
struct DeltaRows {
  void* p;
  int64_t sb, ss, sh;
};

struct DeltaParams {
  DeltaRows q, k, v, o;              // q, k: Hk heads of dk; v, o: H heads of dv
  DeltaRows g, beta;                 // fp32, H scalars a token
  const int* lengths;                // [B] tokens in use, or NULL
  const float* init;                 // [B,H,dk,dv], or NULL
  float* fin;                        // [B,H,dk,dv], or NULL
  float* z;                          // [B,H,N][64][64]
  float* a;                          // [B,H,N][dkp][dkp]
  float* s;                          // [B,H,N][dkp][dvp]
  // the backward's
  DeltaRows dout, dq, dk, dv, dg, dbeta;
  const float* grad_state;           // [B,H,dk,dv], or NULL
  float* grad_init;                  // [B,H,dk,dv], or NULL
  float* d;                          // [B,H,N][dkp][dvp]
  int B, S, H, Hk, dk_, dv_, dkp, dvp, N;
  float scale;
  int vec;                           // rows of q, k, v, o, dout, dq, dk, dv start at multiples of 4 elements
};

// Row b's state is slot b, or slots[b] of a pool of n_slots (state_s elements
// apart); init is read and fin written there (either may be NULL, both may be
// the same memory).
struct DeltaStepParams {
  DeltaRows q, k, v, o, g, beta;
  const float* init;
  float* fin;
  int64_t state_s, n_slots;
  const int64_t* slots;              // [B] or NULL; negative: an idle row
  const int* lengths;                // [B] tokens in use, or NULL
  int B, S, H, Hk, dk_, dv_;
  float scale;
};

hipError_t launch_delta_step(const DeltaStepParams& p, int dtype, hipStream_t stream);
hipError_t launch_delta_fwd(const DeltaParams& p, int dtype, hipStream_t stream);
// part: 2 B S H dk floats where q and k heads are shared.
hipError_t launch_delta_bwd(const DeltaParams& p, float* part, int dtype, hipStream_t stream);
// The chunks' state maps S' = a S + x applied from init, x receiving the state
// before each chunk, fin (or NULL) the last; reverse goes from the last chunk.
hipError_t launch_delta_scan(const DeltaParams& p, const float* a, float* x, const float* init, float* fin,
                             bool reverse, hipStream_t stream);

#ifdef __HIPCC__
namespace delta {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

// A tile in LDS: up to 64 rows of up to 64 floats, 68 apart (four banks a row:
// 16-byte reads of eight consecutive rows touch every bank once).
constexpr int kLd = 68;
constexpr int kTile = 64 * kLd;

__device__ __forceinline__ f32x4 zero4() { return f32x4{0.0f, 0.0f, 0.0f, 0.0f}; }

// acc[c] += A[r0..r0+15][k0..k1) B[k0..k1)[c0+16c..] on the fp32 matrix
// instruction (16x16x4), one wave.  AT: A is stored [k][row]; BT: B is stored
// [column][k]; SC: A's column k is multiplied by sc[k].  k0 and k1 are
// multiples of 16.  Lane group g = lane/16 takes the terms k + 4g .. k + 4g + 3
// of each 16, so that an operand whose k runs along a row is one 16-byte read.
// Result layout: acc[c][i] is row r0 + 4 (lane/16) + i, column c0 + 16 c + lane%16.
template <int CT, bool AT, bool BT, bool SC = false>
__device__ __forceinline__ void mma(f32x4 (&acc)[CT], const float* A, int r0, const float* B, int c0, int k0, int k1,
                                    const float* sc = nullptr) {
  const int l = threadIdx.x & 63, r = l & 15, g = l >> 4;
  for (int k = k0; k < k1; k += 16) {
    f32x4 a, b[CT];
    if (AT) {
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = A[(k + 4 * g + i) * kLd + r0 + r];
    } else {
      a = *reinterpret_cast<const f32x4*>(A + (r0 + r) * kLd + k + 4 * g);
    }
    if (SC) {
      const f32x4 s = *reinterpret_cast<const f32x4*>(sc + k + 4 * g);
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] *= s[i];
    }
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      if (BT) {
        b[c] = *reinterpret_cast<const f32x4*>(B + (c0 + 16 * c + r) * kLd + k + 4 * g);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) b[c][i] = B[(k + 4 * g + i) * kLd + c0 + 16 * c + r];
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < CT; ++c) acc[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[c][i], acc[c], 0, 0, 0);
  }
}

template <int CT>
__device__ __forceinline__ void clear(f32x4 (&acc)[CT]) {
#pragma unroll
  for (int c = 0; c < CT; ++c) acc[c] = zero4();
}

// Row and column of element i of a result's tile c.
__device__ __forceinline__ int out_row(int r0, int i) { return r0 + 4 * ((threadIdx.x & 63) >> 4) + i; }
__device__ __forceinline__ int out_col(int c0, int c) { return c0 + 16 * c + (threadIdx.x & 15); }

template <int CT>
__device__ __forceinline__ void put(float* dst, const f32x4 (&acc)[CT], int r0, int c0) {
#pragma unroll
  for (int c = 0; c < CT; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) dst[out_row(r0, i) * kLd + out_col(c0, c)] = acc[c][i];
}

template <int CT>
__device__ __forceinline__ void get(f32x4 (&acc)[CT], const float* src, int r0, int c0) {
#pragma unroll
  for (int c = 0; c < CT; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[c][i] = src[out_row(r0, i) * kLd + out_col(c0, c)];
}

__device__ __forceinline__ f32x4 load4(const float* p) { return *reinterpret_cast<const f32x4*>(p); }
__device__ __forceinline__ f32x4 load4(const __bf16* p) {
  const bf16x4 v = *reinterpret_cast<const bf16x4*>(p);
  return f32x4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
}

// rows x cols of src (rows `stride` elements apart) into a tile, zeros up to 64
// rows and `width` columns (a multiple of 16).  vec: cols and every row's start
// are multiples of 4 elements.
template <int NT, typename T>
__device__ __forceinline__ void load_tile(float* dst, const T* src, int64_t stride, int rows, int cols, int width,
                                          bool vec) {
  const int quads = width >> 2;
  for (int e = threadIdx.x; e < 64 * quads; e += NT) {
    const int row = e / quads, col = 4 * (e - row * quads);
    f32x4 v = zero4();
    if (row < rows) {
      const T* p = src + row * stride + col;
      if (vec) {
        if (col < cols) v = load4(p);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (col + i < cols) v[i] = (float)p[i];
      }
    }
    *reinterpret_cast<f32x4*>(dst + row * kLd + col) = v;
  }
}

// The same from a workspace matrix of fp32 rows, whole quads.
template <int NT>
__device__ __forceinline__ void load_ws(float* dst, const float* src, int ld, int rows, int width) {
  const int quads = width >> 2;
  for (int e = threadIdx.x; e < rows * quads; e += NT) {
    const int row = e / quads, col = 4 * (e - row * quads);
    *reinterpret_cast<f32x4*>(dst + row * kLd + col) = load4(src + (int64_t)row * ld + col);
  }
}

// The decays of a chunk.  G, the running sum of g, is held as a pair of floats
// (hi + lo, from a double sum), so that differences of long sums keep their
// digits; g below -200 counts as -200, where e^g is 0 in fp32 already (and
// -inf would make the differences NaN).
struct Gates {
  float hi[64], lo[64];
  float beta[64];
  float gam[64];      // e^G
  float end[64];      // e^(G_last - G)
  float bgam[64];     // beta e^G
  float last;         // e^G_last
};

// By the first wave; the caller synchronises.  Tokens past `rows`: g = beta = 0.
__device__ __forceinline__ void load_gates(Gates* s, const DeltaRows& g, const DeltaRows& beta, int64_t b, int64_t t0,
                                           int64_t h, int rows) {
  const int t = threadIdx.x;
  if (t >= 64) return;
  float gv = 0.0f, bv = 0.0f;
  if (t < rows) {
    gv = static_cast<const float*>(g.p)[b * g.sb + (t0 + t) * g.ss + h * g.sh];
    bv = static_cast<const float*>(beta.p)[b * beta.sb + (t0 + t) * beta.ss + h * beta.sh];
    if (gv < -200.0f) gv = -200.0f;
  }
  double G = gv;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double up = __shfl_up(G, o);
    if (t >= o) G += up;
  }
  const double all = __shfl(G, 63);
  const float hi = (float)G;
  s->hi[t] = hi;
  s->lo[t] = (float)(G - hi);
  s->beta[t] = bv;
  const float gam = expf(hi) * (1.0f + (float)(G - hi));
  s->gam[t] = gam;
  s->bgam[t] = bv * gam;
  s->end[t] = expf((float)(all - G));
  if (t == 63) s->last = gam;
}

// e^(G_i - G_j)
__device__ __forceinline__ float decay_between(const Gates& s, int i, int j) {
  return expf((s.hi[i] - s.hi[j]) + (s.lo[i] - s.lo[j]));
}

// (b, h, chunk, tokens in use) of a workgroup's chunk.
struct At {
  int b, h, n, bh;
  int64_t t0;
  int rows;          // tokens of this chunk in use
  int tokens;        // of the row
};
__device__ __forceinline__ At chunk_at(const DeltaParams& p, int64_t id) {
  At w;
  w.n = (int)(id % p.N);
  w.bh = (int)(id / p.N);
  w.b = w.bh / p.H;
  w.h = w.bh - w.b * p.H;
  w.t0 = (int64_t)w.n * kDeltaChunk;
  w.tokens = p.lengths ? min(max(p.lengths[w.b], 0), p.S) : p.S;
  w.rows = (int)min((int64_t)kDeltaChunk, max((int64_t)0, w.tokens - w.t0));
  return w;
}

template <typename T>
__device__ __forceinline__ T* row_ptr(const DeltaRows& r, int64_t b, int64_t t, int64_t h) {
  return static_cast<T*>(r.p) + b * r.sb + t * r.ss + h * r.sh;
}

}  // namespace delta
#endif

}  // namespace osm
