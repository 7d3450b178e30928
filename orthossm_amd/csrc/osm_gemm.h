// A tile of a product of two bf16 matrices with contiguous rows, C = A B^T, on
// gfx950's matrix instruction: what the vocabulary's cross entropy is built on.
//
// A workgroup forms TM x TN of C.  64 columns of both operands' rows at a time go
// from memory to LDS without passing through registers, into one of two buffers
// while the other is multiplied.  A row's 16-byte units lie in LDS at their index
// xor half the row's, so that the 32 rows of a matrix instruction are read from
// different banks; the order is made by the addresses that are read from memory.
// An fp32 operand is three bf16 matrices whose sum it is (its parts), and the
// product the sum of the six products of parts that are not below 2^-24.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace osm {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kStep = 64;        // columns of a step
constexpr int kUnits = kStep / 8;

struct GemmSide {
  const __bf16* p;               // rows ld apart, a multiple of 8; 16-byte aligned
  int64_t ld, part;              // elements from row to row (below 2^21), from part to part
  int rows;                      // rows to read (past them: the last one again)
};

template <int TM_, int TN_, int WM_, int WN_>
struct GemmTile {
  static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_;   // tile; waves along each
  static constexpr int kThreads = 64 * WM * WN;
  static constexpr int FM = TM / WM / 32, FN = TN / WN / 32;     // 32 x 32 squares of a wave
  static constexpr int kBuffer = (TM + TN) * kStep;              // elements of a buffer
  static constexpr int kLds = 2 * kBuffer;
  static_assert(TM * kUnits % kThreads == 0 && TN * kUnits % kThreads == 0, "whole loads");
};

// Where a thread's accumulators lie in C's tile: row(i) of column col, i in [0, 16).
template <class G>
struct GemmPlace {
  int m, n, lane;   // first row and column of the wave
  __device__ __forceinline__ GemmPlace() {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    m = wave % G::WM * (G::TM / G::WM);
    n = wave / G::WM * (G::TN / G::WN);
    lane = threadIdx.x & 63;
  }
  // accumulator i of square (fm, fn)
  __device__ __forceinline__ int row(int fm, int i) const { return m + 32 * fm + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3); }
  __device__ __forceinline__ int col(int fn) const { return n + 32 * fn + (lane & 31); }
};

__device__ __forceinline__ void to_lds(const __bf16* from, __bf16* to) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, (__attribute__((address_space(3))) void*)to, 16,
                                   0, 0);
}

// acc = the rows from m0 of A times the rows from n0 of B over `steps` steps of
// columns from column k0 (a multiple of kStep).  parts: 1, or 3 for each side.
template <class G>
__device__ __forceinline__ void gemm(const GemmSide& A, const GemmSide& B, int m0, int n0, int64_t k0, int steps, int parts,
                                     __bf16* lds, f32x16 (&acc)[G::FM][G::FN]) {
  constexpr int NA = G::TM * kUnits / G::kThreads, NB = G::TN * kUnits / G::kThreads;
  const GemmPlace<G> q;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int oa[NA], ob[NB];   // elements from the first row, column k0
#pragma unroll
  for (int i = 0; i < NA; ++i) {
    const int u = tid + i * G::kThreads, r = u / kUnits, c = (u % kUnits) ^ ((r >> 1) & 7);
    oa[i] = min(r, A.rows - 1 - m0) * (int)A.ld + 8 * c;
  }
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    const int u = tid + i * G::kThreads, r = u / kUnits, c = (u % kUnits) ^ ((r >> 1) & 7);
    ob[i] = min(r, B.rows - 1 - n0) * (int)B.ld + 8 * c;
  }
  const __bf16* const a0 = A.p + m0 * A.ld + k0;
  const __bf16* const b0 = B.p + n0 * B.ld + k0;
  const int segments = parts == 1 ? 1 : 6, total = steps * segments;
  // (parts i of A and j of B in order: 2 0, 1 1, 0 2, 1 0, 0 1, 0 0, the small ones first)
  int seg = 0, at = 0;
  const __bf16 *pa, *pb;
  auto point = [&] {
    const int i = segments == 1 ? 0 : (0x001012 >> (4 * seg)) & 15, j = segments == 1 ? 0 : (0x010210 >> (4 * seg)) & 15;
    pa = a0 + i * A.part;
    pb = b0 + j * B.part;
  };
  point();
  auto fetch = [&](int buf) {
    __bf16* const to = lds + buf * G::kBuffer + wave * 512;
#pragma unroll
    for (int i = 0; i < NA; ++i) to_lds(pa + oa[i], to + i * G::kThreads * 8);
#pragma unroll
    for (int i = 0; i < NB; ++i) to_lds(pb + ob[i], to + G::TM * kStep + i * G::kThreads * 8);
    pa += kStep;
    pb += kStep;
    if (++at == steps) {
      at = 0;
      ++seg;
      point();
    }
  };
#pragma unroll
  for (int i = 0; i < G::FM; ++i)
#pragma unroll
    for (int j = 0; j < G::FN; ++j) acc[i][j] = (f32x16)0.0f;
  // a lane's row of a square and its unit in each half step
  const int r = q.lane & 31, half = q.lane >> 5, x = (r >> 1) & 7;   // (squares start at multiples of 32 rows: x is the same)
  if (total > 0) fetch(0);
  for (int t = 0; t < total; ++t) {
    __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0): this step's units are in LDS
    __syncthreads();                      // everyone's are, and the other buffer has been read
    if (t + 1 < total) fetch((t + 1) & 1);
    const __bf16* const la = lds + (t & 1) * G::kBuffer;
    const __bf16* const lb = la + G::TM * kStep;
#pragma unroll
    for (int s = 0; s < kStep / 16; ++s) {
      const int unit = ((2 * s + half) ^ x) * 8;
      bf16x8 fa[G::FM], fb[G::FN];
#pragma unroll
      for (int i = 0; i < G::FM; ++i) fa[i] = *reinterpret_cast<const bf16x8*>(la + (q.m + 32 * i + r) * kStep + unit);
#pragma unroll
      for (int j = 0; j < G::FN; ++j) fb[j] = *reinterpret_cast<const bf16x8*>(lb + (q.n + 32 * j + r) * kStep + unit);
#pragma unroll
      for (int i = 0; i < G::FM; ++i)
#pragma unroll
        for (int j = 0; j < G::FN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[i], fb[j], acc[i][j], 0, 0, 0);
    }
  }
  __syncthreads();   // the buffers are free
}

}  // namespace osm
