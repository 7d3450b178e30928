// A tile of a product of two bf16 matrices on gfx950's matrix instruction, C[n][m] =
// sum_k A(m, k) B(n, k): what the vocabulary's cross entropy is built on.
//
// Each operand lies by rows (a row holds the k of one m or n) or by columns (a row
// holds the m or n of one k).  A workgroup forms TM x TN of C.  64 k (32 of operands in
// parts) of both operands at a time go from memory to LDS without passing through
// registers, into one buffer while another is multiplied.  By rows, a row's 16-byte units
// lie in LDS at their index xor half the row's, so that the 32 rows of a matrix
// instruction are read from different banks; by columns, a row's 32-byte units lie at
// theirs xor the row's, so that the 4 rows of a transposing read are.  The order is made by
// the addresses that are read from memory.
//
// An fp32 operand is three bf16 matrices whose sum it is (its parts), and the product the
// sum of the six products of parts that are not below 2^-24: the product of the first
// parts, and in accumulators of their own the five small ones.  All parts of a step lie in
// LDS together: they come from memory and are read once for the six products (5003 x 981 x
// 448: 36 us; with a walk over k for each product 49).
//
// What bounds it: the matrix instructions, half of the time (50176 x 8192 x 1024 in tiles of
// 256 x 256: 680 us, 1238 TFLOP/s, by columns both ways 1170; 16384 x 4096 x 1024 of three
// parts 1172).  128 KB of LDS leave no room for a third buffer; to read a step's first part
// across the barrier, while the last of the step before is multiplied, gains 1%.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace osm {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kStep = 64;        // k come in multiples of this

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

struct GemmSide {
  const __bf16* p;               // rows ld apart, a multiple of 8; 16-byte aligned
  int64_t ld, part;              // elements from row to row (below 2^21), from part to part
  int rows;                      // rows to read (past them: the last one again)
  int cols;                      // by columns: elements of a row to read, a multiple of 8 (past them: the last ones again)
};

template <int TM_, int TN_, int WM_, int WN_, int PARTS_ = 1, int ST_ = 2>
struct GemmTile {
  static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_;   // tile; waves along each
  static constexpr int PARTS = PARTS_, ST = ST_;                 // of an operand; buffers
  static constexpr int KS = PARTS == 1 ? 64 : 32;                // k of a step
  static constexpr int kThreads = 64 * WM * WN;
  static constexpr bool kFew = PARTS == 1 && TM < 256;           // for few tokens too
  static constexpr int FM = TM / WM / 32, FN = TN / WN / 32;     // 32 x 32 squares of a wave
  static constexpr int kBuffer = PARTS * (TM + TN) * KS;         // elements of a buffer: A's parts, then B's
  static constexpr int kLds = ST * kBuffer;
  static constexpr int kLoads = kBuffer / 8 / kThreads;          // of a thread and step
  static_assert(TM * KS / 8 % kThreads == 0 && TN * KS / 8 % kThreads == 0 && kStep % KS == 0, "whole loads and steps");
};

// Waits until at most N of this wave's loads are on their way.
template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N < 64, "6 bits");
  __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | (N >> 4) << 14);
}

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

// 16 bytes a lane from memory to LDS, to the 1024 bytes from `to` (the same in every lane)
// on in the order of the lanes.  It has no result to wait for: who reads them waits for
// vmcnt himself.  (In place of the compiler's builtin, ahead of whose effects it would
// wait at the next transposing read, which is of the other buffer.)  What the compiler may
// hold in M0 it sets again: the register is declared, though not one that it allocates, of
// which it would warn.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void to_lds(const __bf16* from, unsigned to) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(to) : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ unsigned lds_address(const __bf16* p) {
  return (unsigned)(uintptr_t)(const __attribute__((address_space(3))) __bf16*)p;
}

// One operand of a tile, T of its m or n: where a thread's share of a step comes from, and
// where a lane's share of a matrix instruction lies in LDS.
template <class G, int T, bool COLS>
struct GemmOperand {
  static constexpr int KS = G::KS, kRow = COLS ? T : KS, kRowUnits = kRow / 8;   // elements, 16-byte units of a row in LDS
  static constexpr int N = T * KS / 8 / G::kThreads;
  // (rows of 128 bytes: two of them go through the banks; of 64 bytes: four)
  static __device__ __forceinline__ int turn(int row) { return KS == 64 ? row >> 1 & 7 : row >> 2 & 3; }
  int from[N];             // elements from the step's first
  const __bf16* first;     // the next step's
  int64_t ld, part;
  int rows, k;             // by columns: rows in all, and ahead of the step

  static __device__ __forceinline__ int row_of(int i) { return ((int)threadIdx.x + i * G::kThreads) / kRowUnits; }
  static __device__ __forceinline__ int col_of(int i) {
    const int u = (int)threadIdx.x + i * G::kThreads, r = u / kRowUnits, c = u % kRowUnits;
    return 8 * (COLS ? (c ^ ((r & 3) << 1)) : (c ^ turn(r)));
  }
  __device__ __forceinline__ GemmOperand(const GemmSide& s, int m0, int64_t k0) {
    ld = s.ld;
    part = s.part;
    rows = s.rows;
    k = (int)k0;
    first = s.p + (COLS ? k0 * ld + m0 : m0 * ld + k0);
#pragma unroll
    for (int i = 0; i < N; ++i)
      from[i] = COLS ? row_of(i) * (int)ld + min(col_of(i), s.cols - 8 - m0) : min(row_of(i), rows - 1 - m0) * (int)ld + col_of(i);
  }
  // The next step to LDS.
  __device__ __forceinline__ void fetch(unsigned to) {
    to += __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 1024;
    const bool whole = !COLS || k + KS <= rows;
#pragma unroll
    for (int q = 0; q < G::PARTS; ++q) {
      const __bf16* const at = first + q * part;
      const unsigned there = to + q * T * KS * 2;
      if (whole) {
#pragma unroll
        for (int i = 0; i < N; ++i) to_lds(at + from[i], there + i * G::kThreads * 16);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int r = row_of(i), over = max(r + k - (rows - 1), 0);
          to_lds(at + from[i] - (int64_t)over * ld, there + i * G::kThreads * 16);
        }
      }
    }
    first += COLS ? KS * ld : KS;
    k += KS;
  }
  // A lane's 8 elements of the 32 from `m` on, in the s-th 16 k of the step.
  static __device__ __forceinline__ bf16x8 read(const __bf16* lds, int m, int s, int lane) {
    if constexpr (!COLS) {
      const int r = lane & 31;
      return *reinterpret_cast<const bf16x8*>(lds + (m + r) * KS + (((2 * s + (lane >> 5)) ^ turn(r)) * 8));
    } else {
      // (a group of 16 lanes reads 4 rows of 16 elements and gets them by columns)
      const int i = lane & 15, g = lane >> 4, r = 16 * s + 8 * (g >> 1) + (i >> 2);
      const __bf16* const p = lds + r * kRow + (((m >> 4) + (g & 1)) ^ (i >> 2)) * 16 + (i & 3) * 4;
      typedef __attribute__((address_space(3))) i16x4* Lds;
      const bf16x4 lo = __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(p)));
      const bf16x4 hi = __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(p + 4 * kRow)));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
};

template <class G>
__device__ __forceinline__ void zero(f32x16 (&acc)[G::FM][G::FN]) {
#pragma unroll
  for (int i = 0; i < G::FM; ++i)
#pragma unroll
    for (int j = 0; j < G::FN; ++j) acc[i][j] = (f32x16)0.0f;
}

// acc += the m from m0 of A times the n from n0 of B over n_steps times kStep k from k0 on (a
// multiple of kStep).
template <class G, bool ACOLS, bool BCOLS>
__device__ __forceinline__ void gemm(const GemmSide& A, const GemmSide& B, int m0, int n0, int64_t k0, int n_steps, __bf16* lds,
                                     f32x16 (&acc)[G::FM][G::FN]) {
  using OA = GemmOperand<G, G::TM, ACOLS>;
  using OB = GemmOperand<G, G::TN, BCOLS>;
  constexpr int P = G::PARTS;
  const GemmPlace<G> q;
  OA a(A, m0, k0);
  OB b(B, n0, k0);
  const int steps = n_steps * (kStep / G::KS);
  const unsigned base = __builtin_amdgcn_readfirstlane(lds_address(lds));
  auto fetch = [&](int buf) {
    const unsigned to = base + buf * G::kBuffer * 2;
    a.fetch(to);
    b.fetch(to + P * G::TM * G::KS * 2);
  };
  f32x16 small[P == 1 ? 1 : G::FM][G::FN];
  if constexpr (P > 1) zero<G>(small);
  // Step t is multiplied while the ST - 1 after it are on their way; the last of those goes
  // where step t - 1 was, which everyone has read by the barrier.
#pragma unroll
  for (int t = 0; t < G::ST - 1; ++t)
    if (t < steps) fetch(t);
  int buf = 0;
  for (int t = 0; t < steps; ++t) {
    if (t + G::ST - 2 < steps)
      wait_loads<(G::ST - 2) * G::kLoads>();
    else
      wait_loads<0>();
    __syncthreads();
    if (t + G::ST - 1 < steps) fetch(buf == 0 ? G::ST - 1 : buf - 1);
    const __bf16* const la = lds + buf * G::kBuffer;
    const __bf16* const lb = la + P * G::TM * G::KS;
    buf = buf == G::ST - 1 ? 0 : buf + 1;
    // By rows, what the next 16 k take is read while these are multiplied, a read after each
    // matrix instruction (50176 x 8192 x 1024: 735 us without, 695 with; transposing reads,
    // twice as many, are better left to the compiler: 231 and 237 us for 1024 x 16384 x 8192).
    constexpr bool kAhead = !ACOLS && !BCOLS;
    constexpr int kParts = G::KS / 16, kHeld = kAhead ? 2 : 1;
    bf16x8 fa[kHeld][P][G::FM], fb[kHeld][P][G::FN];
    auto read = [&](int s) {
#pragma unroll
      for (int p = 0; p < P; ++p) {
#pragma unroll
        for (int i = 0; i < G::FM; ++i) fa[s % kHeld][p][i] = OA::read(la + p * G::TM * G::KS, q.m + 32 * i, s, q.lane);
#pragma unroll
        for (int j = 0; j < G::FN; ++j) fb[s % kHeld][p][j] = OB::read(lb + p * G::TN * G::KS, q.n + 32 * j, s, q.lane);
      }
    };
    if (kAhead) read(0);
#pragma unroll
    for (int s = 0; s < kParts; ++s) {
      if (!kAhead)
        read(s);
      else if (s + 1 < kParts)
        read(s + 1);
      auto multiply = [&](int pa, int pb, f32x16 (&to)[G::FM][G::FN]) {
#pragma unroll
        for (int i = 0; i < G::FM; ++i)
#pragma unroll
          for (int j = 0; j < G::FN; ++j)
            to[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[s % kHeld][pa][i], fb[s % kHeld][pb][j], to[i][j], 0, 0, 0);
      };
      if constexpr (P > 1) {
        multiply(2, 0, small);
        multiply(0, 2, small);
        multiply(1, 1, small);
        multiply(1, 0, small);
        multiply(0, 1, small);
      }
      multiply(0, 0, acc);
      if constexpr (kAhead) {
#pragma unroll
        for (int i = 0; i < G::FM * G::FN * (P > 1 ? 6 : 1); ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);   // a matrix instruction
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);   // an LDS read
        }
      }
    }
  }
  // (an infinite operand is so in its first part, and its other products are none)
  if constexpr (P > 1)
#pragma unroll
    for (int i = 0; i < G::FM; ++i)
#pragma unroll
      for (int j = 0; j < G::FN; ++j)
#pragma unroll
        for (int k = 0; k < 16; ++k)
          if (__builtin_fabsf(acc[i][j][k]) < __builtin_inff()) acc[i][j][k] += small[i][j][k];
  __syncthreads();   // the buffers are free
}

}  // namespace osm
