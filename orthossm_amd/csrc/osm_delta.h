// Parameters of the gated delta rule's kernels (osm_delta.hip,
// osm_delta_bwd.hip) and the tile products both are built from.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "osm_wide_store.h"

namespace osm {

constexpr int kDeltaChunk = 64;      // tokens a chunk
constexpr int kDeltaMaxDk = 128;     // rows of the state
constexpr int kDeltaSlice = 16;      // columns of the state a scan workgroup, or a wave of a walk, holds
constexpr int kGateFloats = 320;     // a chunk's gates (delta::make_gates)
constexpr int kZFloats = 32 * 32 + 32 * 64;   // a chunk's Z: rows 0-31 by 32 columns, rows 32-63 by 64

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
  float* z;                          // [B,H,N][kZFloats]
  float* gates;                      // [B,H,N][kGateFloats]
  float* s;                          // [B,H,N][dkp][dvp] states before the chunks, or NULL
  float* a;                          // maps of the segments [B,H,segs][dkp][dkp]
  float* x;                          // and what they add, then the states before them [B,H,segs][dkp][dvp]
  // the backward's
  DeltaRows dout, dq, dk, dv, dg, dbeta;
  const float* grad_state;           // [B,H,dk,dv], or NULL
  float* grad_init;                  // [B,H,dk,dv], or NULL
  float* d;                          // [B,H,N][dkp][dvp]
  int B, S, H, Hk, dk_, dv_, dkp, dvp, N;   // dkp: dk up to a multiple of 32, dvp: dv of 16, N: chunks of a row
  int seg, segs;                     // chunks a segment, segments a row
  float scale;
  int vec;                           // q, k, v and dout are whole multiples of so many elements, strides and all (4, 2, 1)
  int out_vec;                       // dq's and dk's rows start at multiples of 4 elements
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

int delta_segment(int64_t heads, int64_t chunks);
hipError_t launch_delta_step(const DeltaStepParams& p, int dtype, hipStream_t stream);
hipError_t launch_delta_fwd(const DeltaParams& p, int dtype, hipStream_t stream);
// part: 2 B S H dk floats where q and k heads are shared.
hipError_t launch_delta_bwd(const DeltaParams& p, float* part, int dtype, hipStream_t stream);
// The state maps S' = a S + x of n spans of `span` tokens a row applied from init,
// x receiving the state before each span; reverse goes from the last span.
hipError_t launch_delta_scan(const DeltaParams& p, const float* a, float* x, const float* init, int n, int span,
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

// Row and first column of the four elements `quad` of a stored Z.
__device__ __forceinline__ int z_row(int quad) { return quad < 256 ? quad >> 3 : 32 + ((quad - 256) >> 4); }
__device__ __forceinline__ int z_quad(int quad) { return quad < 256 ? quad & 7 : (quad - 256) & 15; }

// A stored Z into a tile.
template <int NT>
__device__ __forceinline__ void load_z(float* dst, const float* src) {
  for (int e = threadIdx.x; e < kZFloats / 4; e += NT)
    *reinterpret_cast<f32x4*>(dst + z_row(e) * kLd + 4 * z_quad(e)) = load4(src + 4 * e);
  for (int e = threadIdx.x; e < 256; e += NT) *reinterpret_cast<f32x4*>(dst + (e >> 3) * kLd + 32 + 4 * (e & 7)) = zero4();
}

// A workspace matrix of fp32 rows, whole quads, into a tile.
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

// ---- bf16 parts of fp32 numbers ----

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// bf16 numbers that hold one of T.
template <typename T>
constexpr int kParts = sizeof(T) == 4 ? 3 : 1;

// a and b as the sums of N bf16 numbers each, packed: the nearest, then the
// nearest to what is left, and again (three hold all 24 bits).  What is left,
// x - part, is exact, and one instruction as a dot product of the packed pair.
template <int N>
__device__ __forceinline__ void split2(unsigned (&part)[N], float a, float b) {
  // (-1, 0) and (0, -1), as values that the compiler does not fold: it writes the
  // first as the instruction's inline -1.0, which the hardware reads as an fp32
  // number, that is as (0, -1).
  unsigned first, second;
  asm("s_mov_b32 %0, 0xbf80" : "=s"(first));
  asm("s_mov_b32 %0, 0xbf800000" : "=s"(second));
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const bf16x2 h = __builtin_convertvector(f32x2{a, b}, bf16x2);
    part[k] = __builtin_bit_cast(unsigned, h);
    if (k < N - 1) {
      a = __builtin_amdgcn_fdot2_f32_bf16(h, __builtin_bit_cast(bf16x2, first), a, false);
      b = __builtin_amdgcn_fdot2_f32_bf16(h, __builtin_bit_cast(bf16x2, second), b, false);
    }
  }
}

template <int N>
__device__ __forceinline__ void split4(u32x2 (&part)[N], f32x4 v) {
  unsigned lo[N], hi[N];
  split2<N>(lo, v[0], v[1]);
  split2<N>(hi, v[2], v[3]);
#pragma unroll
  for (int k = 0; k < N; ++k) part[k] = u32x2{lo[k], hi[k]};
}

// Two result tiles, rows 16 apart, as the second operand of a product over
// their 32 rows.
template <int N>
__device__ __forceinline__ void split_pair(u32x4 (&part)[N], f32x4 a, f32x4 b) {
  u32x2 pa[N], pb[N];
  split4<N>(pa, a);
  split4<N>(pb, b);
#pragma unroll
  for (int k = 0; k < N; ++k) part[k] = u32x4{pa[k][0], pa[k][1], pb[k][0], pb[k][1]};
}

// The terms of a product's 32 are kept in the order in which a pair of result
// tiles holds them: place 8 g + 4 h + i is term 16 h + 4 g + i.  Place of the
// four terms 4 q .. 4 q + 3 along a row:
__device__ __forceinline__ int place4(int q) { return 32 * (q >> 3) + 8 * (q & 3) + 4 * ((q >> 2) & 1); }

// The parts of 8 terms at `at` of matrices `stride` elements apart.
template <int NP>
__device__ __forceinline__ void read_parts(u32x4 (&f)[NP], const unsigned short* m, int stride, int at) {
#pragma unroll
  for (int k = 0; k < NP; ++k) f[k] = *reinterpret_cast<const u32x4*>(m + k * stride + at);
}

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// acc += A B over 32 terms, the smaller products first; products of parts i and
// j with i + j > ORDER (of order 2^(-8 ORDER - 8) and below) are left out.
template <int NB, int ORDER, int NA, int N>
__device__ __forceinline__ void mul(f32x4& acc, const u32x4 (&a)[NA], const u32x4 (&b)[N]) {
  static_assert(NB <= N, "no more parts than there are");
#pragma unroll
  for (int sum = ORDER; sum >= 0; --sum)
#pragma unroll
    for (int i = 0; i <= sum; ++i)
      if (i < NA && sum - i < NB) acc = mfma(a[i], b[sum - i], acc);
}

// COUNT products in turn: at(i) is where the parts of the i-th first operand are
// in LDS, go(i, parts) its matrix instructions.  Operands are read DEPTH products
// ahead: left to itself the compiler reads each right before its use, and a wave
// then waits for LDS as long again as it computes.
template <int NA, int DEPTH, int COUNT, typename At, typename Go>
__device__ __forceinline__ void products(int stride, At at, Go go) {
  constexpr int kStay = 0;
  u32x4 a[DEPTH + 1][NA];
#pragma unroll
  for (int i = 0; i < DEPTH && i < COUNT; ++i) read_parts<NA>(a[i], at(i), stride, 0);
#pragma unroll
  for (int i = 0; i < COUNT; ++i) {
    if (i + DEPTH < COUNT) read_parts<NA>(a[(i + DEPTH) % (DEPTH + 1)], at(i + DEPTH), stride, 0);
    __builtin_amdgcn_sched_barrier(kStay);
    go(i, a[i % (DEPTH + 1)]);
    __builtin_amdgcn_sched_barrier(kStay);
  }
}

__device__ __forceinline__ void store4(float* p, f32x4 v) {
  *reinterpret_cast<f32x4*>(p) = v;
  wide_store_wait();
}

// Memory through buffer descriptors: an access past the extent reads zeros and
// drops stores.  A descriptor of a chunk's rows ends with its last row in use, so
// rows past it need no test (a row's stride is at least its length: the entry
// points see to it); a column outside the tensor has kOut as its offset.  The
// row's offset is added by the scalar operand: one address register for all.
typedef __amdgpu_buffer_rsrc_t Rsrc;
constexpr unsigned kOut = 0x80000000u;
__device__ __forceinline__ Rsrc make_rsrc(const void* base, unsigned extent = 0x7fffffffu) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, (int)extent, 0x00020000);
}
// `rows` rows of `cols` elements of T.
template <typename T>
__device__ __forceinline__ Rsrc rows_rsrc(const void* base, int64_t stride, int rows, int cols) {
  return make_rsrc(base, rows > 0 ? ((unsigned)(rows - 1) * (unsigned)stride + cols) * (unsigned)sizeof(T) : 0);
}

// An element as it comes, in a register of its own, and its value.
template <typename T>
__device__ __forceinline__ unsigned load_raw(Rsrc r, unsigned at, unsigned row = 0) {
  if constexpr (sizeof(T) == 4)
    return __builtin_amdgcn_raw_buffer_load_b32(r, at, row, 0);
  else
    return __builtin_amdgcn_raw_buffer_load_b16(r, at, row, 0);
}
template <typename T>
__device__ __forceinline__ float raw_value(unsigned v) {
  return __uint_as_float(sizeof(T) == 4 ? v : v << 16);
}
template <typename T>
__device__ __forceinline__ void store_one(Rsrc r, unsigned at, unsigned row, float v) {
  if constexpr (sizeof(T) == 4)
    __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), r, at, row, 0);
  else
    __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, (__bf16)v), r, at, row, 0);
}

// 64 rows of 32 KS columns of q or k in the registers of NT threads: 4x4 blocks,
// the columns' blocks of a row in consecutive threads.
template <typename T, int KS, int NT>
struct Block {
  static constexpr int kQuads = 8 * KS, kBlocks = (16 * kQuads + NT - 1) / NT;
  static constexpr bool kAll = 16 * kQuads % NT == 0;
  static constexpr int NP = kParts<T>;
  typedef typename std::conditional<sizeof(T) == 4, f32x4, bf16x4>::type Quad;
  Quad v[kBlocks][4];

  __device__ __forceinline__ void load(const T* src, int64_t stride, int rows, int cols, int vec) {
    const Rsrc rs = rows_rsrc<T>(src, stride, rows, cols);
    const unsigned es = sizeof(T), row_bytes = (unsigned)stride * es;
#pragma unroll
    for (int n = 0; n < kBlocks; ++n) {
      const int e = threadIdx.x + n * NT, q = e % kQuads, r = 4 * (e / kQuads);
      const unsigned at = (kAll || e < 16 * kQuads) && 4 * q < cols ? r * row_bytes + 4 * q * es : kOut;
      if (vec == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (sizeof(T) == 4)
            v[n][i] = __builtin_bit_cast(Quad, __builtin_amdgcn_raw_buffer_load_b128(rs, at, i * row_bytes, 0));
          else
            v[n][i] = __builtin_bit_cast(Quad, __builtin_amdgcn_raw_buffer_load_b64(rs, at, i * row_bytes, 0));
        }
      } else if (sizeof(T) == 2 && vec == 2) {
        const unsigned at2 = 4 * q + 2 < cols ? at + 2 * es : kOut;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if constexpr (sizeof(T) == 2)
            v[n][i] = __builtin_bit_cast(Quad, u32x2{__builtin_amdgcn_raw_buffer_load_b32(rs, at, i * row_bytes, 0),
                                                     __builtin_amdgcn_raw_buffer_load_b32(rs, at2, i * row_bytes, 0)});
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            v[n][i][k] = (T)raw_value<T>(load_raw<T>(rs, 4 * q + k < cols ? at + k * es : kOut, i * row_bytes));
      }
    }
  }
  // rows LD elements apart, the parts `stride`
  template <int LD>
  __device__ __forceinline__ void put_rows(unsigned short* dst, int stride) const {
#pragma unroll
    for (int n = 0; n < kBlocks; ++n) {
      const int e = threadIdx.x + n * NT, q = e % kQuads, r = 4 * (e / kQuads);
      if (kAll || e < 16 * kQuads)
#pragma unroll
        for (int i = 0; i < 4; ++i) put(dst + (r + i) * LD + place4(q), stride, v[n][i]);
    }
  }
  // columns LD elements apart
  template <int LD>
  __device__ __forceinline__ void put_columns(unsigned short* dst, int stride) const {
#pragma unroll
    for (int n = 0; n < kBlocks; ++n) {
      const int e = threadIdx.x + n * NT, q = e % kQuads, r = e / kQuads;
      if (kAll || e < 16 * kQuads)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          put(dst + (4 * q + k) * LD + place4(r), stride, Quad{v[n][0][k], v[n][1][k], v[n][2][k], v[n][3][k]});
    }
  }

 private:
  static __device__ __forceinline__ void put(unsigned short* dst, int stride, Quad x) {
    if constexpr (NP == 1) {
      *reinterpret_cast<u32x2*>(dst) = __builtin_bit_cast(u32x2, x);
    } else {
      u32x2 part[3];
      split4<3>(part, x);
#pragma unroll
      for (int k = 0; k < 3; ++k) *reinterpret_cast<u32x2*>(dst + k * stride) = part[k];
    }
  }
};

// A chunk's gates as the solve leaves them, 64 floats each.  hi + lo is G in
// units of log 2, from a double sum, so that differences of long sums keep their
// digits; g below -200 counts as -200, where e^g is 0 in fp32 already (and -inf
// would make the differences NaN).
constexpr int kHi = 0, kLo = 64, kBeta = 128, kGam = 192, kEnd = 256;   // .., beta, e^G, e^(G_last - G)

// By the first wave; the caller synchronises.  Tokens past `rows`: g = beta = 0.
__device__ __forceinline__ void make_gates(float* gt, const DeltaRows& g, const DeltaRows& beta, int64_t b, int64_t t0,
                                           int64_t h, int rows) {
  const int t = threadIdx.x;
  if (t >= 64) return;
  float gv = 0.0f, bv = 0.0f;
  if (t < rows) {
    gv = static_cast<const float*>(g.p)[b * g.sb + (t0 + t) * g.ss + h * g.sh];
    bv = static_cast<const float*>(beta.p)[b * beta.sb + (t0 + t) * beta.ss + h * beta.sh];
    if (gv < -200.0f) gv = -200.0f;
  }
  double G = (double)gv * 1.4426950408889634;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double up = __shfl_up(G, o);
    if (t >= o) G += up;
  }
  const float hi = (float)G, lo = (float)(G - hi);
  gt[kHi + t] = hi;
  gt[kLo + t] = lo;
  gt[kBeta + t] = bv;
  gt[kGam + t] = __builtin_amdgcn_exp2f(hi) * __builtin_fmaf(lo, 0.69314718f, 1.0f);
  gt[kEnd + t] = __builtin_amdgcn_exp2f((float)(__shfl(G, 63) - G));
}

// e^(G_i - G_j)
__device__ __forceinline__ float decay(const float* gt, int i, int j) {
  return __builtin_amdgcn_exp2f((gt[kHi + i] - gt[kHi + j]) + (gt[kLo + i] - gt[kLo + j]));
}

// Rows 0-31 of a lower triangular matrix of the walk have 32 columns, the others
// 64 (plus 8 of padding: 16-byte reads of eight consecutive rows touch every bank
// once).
constexpr int kTri = 32 * 40 + 32 * 72;
__device__ __forceinline__ int tri_at(int row) { return row < 32 ? row * 40 : 1280 + (row - 32) * 72; }

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
