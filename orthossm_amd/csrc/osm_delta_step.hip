// The gated delta rule token by token on gfx950: one token of a served row, or
// a short sequence.  Per state column j, with a = S^T k and b = S^T q of the
// state before the token, everything the token needs is two dot products of
// one read of the state:
//   u = beta (v - e^g a),  o = scale (e^g b + (k.q) u),  S <- e^g S + k u
//
// A workgroup holds 32 columns of a head's state in registers, in row groups of R
// rows that are added through a wave's shuffles and LDS: one barrier a token.  A
// thread holds NC neighbouring columns: four (16-byte accesses) where the rows'
// alignment allows it and there are more than 32 rows, one else (1024 states of 128 by
// 128: 35.7 us with one, 29.5 with four).
// One token is bound by the state's bytes (read and written once, 128-byte
// pieces of rows; the 1024 states at 4.5 TB/s), or by the launch when there are few
// rows (8 states of 64 by 64: 5.2 us).
#include "osm_delta.h"

namespace osm {
namespace {

using namespace delta;

constexpr int kCols = 32, kStepThreads = 256;

template <typename T, int R, int NC>
__global__ void __launch_bounds__(kStepThreads) delta_step_kernel(const DeltaStepParams p) {
  constexpr int kLanes = kCols / NC, kGroups = kStepThreads / kLanes, kRows = R * kGroups;
  __shared__ __attribute__((aligned(16))) float kq[2][2][kRows];
  __shared__ float red[2][4][2 * NC + 1][kLanes];
  const int ncb = (p.dv_ + kCols - 1) / kCols;
  const int tid = threadIdx.x, jl = tid % kLanes, kg = tid / kLanes, wave = tid >> 6;
  const int j = kCols * (int)(blockIdx.x % ncb) + NC * jl, bh = blockIdx.x / ncb;
  const int b = bh / p.H, h = bh - b * p.H, hk = h / (p.H / p.Hk);
  const bool live = j < p.dv_;
  const int64_t slot = p.slots ? p.slots[b] : b;
  typedef float Cols __attribute__((ext_vector_type(NC)));
  T* const o = row_ptr<T>(p.o, b, 0, h) + j;
  auto put_out = [&](int t, Cols v) {
#pragma unroll
    for (int c = 0; c < NC; ++c) o[t * p.o.ss + c] = (T)v[c];
    if (NC * sizeof(T) > 8) wide_store_wait();   // (the compiler makes them one store)
  };
  if (slot < 0 || slot >= p.n_slots) {   // an idle row, or (past the pool) a wrong one: its outputs are NaN
    if (live && kg == 0)
      for (int t = 0; t < p.S; ++t) put_out(t, (Cols)(slot < 0 ? 0.0f : __builtin_nanf("")));
    return;
  }
  const int n = p.lengths ? min(max(p.lengths[b], 0), p.S) : p.S;
  const int64_t at = slot * p.state_s + (int64_t)h * p.dk_ * p.dv_ + j;
  Cols s[R];   // row kg + kGroups i
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = kg + kGroups * i;
    s[i] = p.init && live && row < p.dk_ ? *reinterpret_cast<const Cols*>(p.init + at + (int64_t)row * p.dv_) : (Cols)0.0f;
  }
  // k and q of a token
  auto fetch = [&](int t, int e) {
    const bool is_q = e >= kRows;
    e -= is_q ? kRows : 0;
    return e < p.dk_ ? (float)(is_q ? row_ptr<T>(p.q, b, t, hk) : row_ptr<T>(p.k, b, t, hk))[e] : 0.0f;
  };
  static_assert(2 * kRows <= 2 * kStepThreads, "two values of k and q a thread at most");
  if (n > 0)
    for (int e = tid; e < 2 * kRows; e += kStepThreads) (&kq[0][0][0])[e] = fetch(0, e);
  __syncthreads();
  for (int t = 0; t < n; ++t) {
    const int par = t & 1;
    float next[2];
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (tid + e * kStepThreads < 2 * kRows) next[e] = t + 1 < n ? fetch(t + 1, tid + e * kStepThreads) : 0.0f;
    const float decay = expf(*row_ptr<float>(p.g, b, t, h)), beta = *row_ptr<float>(p.beta, b, t, h);
    Cols v = (Cols)0.0f;
    if (live)
#pragma unroll
      for (int c = 0; c < NC; ++c) v[c] = (float)row_ptr<T>(p.v, b, t, h)[j + c];
    float kk[R], kv = 0.0f;
    Cols sk = (Cols)0.0f, sq = (Cols)0.0f;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const float q = kq[par][1][kg + kGroups * i];
      kk[i] = kq[par][0][kg + kGroups * i];
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        sk[c] = __builtin_fmaf(s[i][c], kk[i], sk[c]);
        sq[c] = __builtin_fmaf(s[i][c], q, sq[c]);
      }
      kv = __builtin_fmaf(q, kk[i], kv);
    }
    float sum[2 * NC + 1];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      sum[c] = sk[c];
      sum[NC + c] = sq[c];
    }
    sum[2 * NC] = kv;
#pragma unroll
    for (int c = 0; c < 2 * NC + 1; ++c) {
#pragma unroll
      for (int m = kLanes; m < 64; m <<= 1) sum[c] += __shfl_xor(sum[c], m);
      if ((tid & 63) < kLanes) red[par][wave][c][jl] = sum[c];
    }
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (tid + e * kStepThreads < 2 * kRows) (&kq[par ^ 1][0][0])[tid + e * kStepThreads] = next[e];
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 2 * NC + 1; ++c)
      sum[c] = (red[par][0][c][jl] + red[par][1][c][jl]) + (red[par][2][c][jl] + red[par][3][c][jl]);
    Cols u;
#pragma unroll
    for (int c = 0; c < NC; ++c) u[c] = beta * (v[c] - decay * sum[c]);
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int c = 0; c < NC; ++c) s[i][c] = __builtin_fmaf(kk[i], u[c], decay * s[i][c]);
    if (live && kg == 0) {
      Cols v_out;
#pragma unroll
      for (int c = 0; c < NC; ++c) v_out[c] = p.scale * __builtin_fmaf(sum[2 * NC], u[c], decay * sum[NC + c]);
      put_out(t, v_out);
    }
  }
  if (live && kg == 0)
    for (int t = n; t < p.S; ++t) put_out(t, (Cols)0.0f);
  if (p.fin && live)
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int row = kg + kGroups * i;
      if (row < p.dk_) {
        *reinterpret_cast<Cols*>(p.fin + at + (int64_t)row * p.dv_) = s[i];
        if (NC == 4) wide_store_wait();
      }
    }
}

template <typename T>
hipError_t step(const DeltaStepParams& p, hipStream_t stream) {
  const dim3 grid((unsigned)((int64_t)p.B * p.H * ((p.dv_ + kCols - 1) / kCols))), block(kStepThreads);
  const bool quads = p.dv_ % 4 == 0 && p.state_s % 4 == 0 && ((uintptr_t)p.init | (uintptr_t)p.fin) % 16 == 0;
  if (quads && p.dk_ > 64)
    hipLaunchKernelGGL((delta_step_kernel<T, 4, 4>), grid, block, 0, stream, p);
  else if (quads && p.dk_ > 32)
    hipLaunchKernelGGL((delta_step_kernel<T, 2, 4>), grid, block, 0, stream, p);
  else if (p.dk_ <= 16)
    hipLaunchKernelGGL((delta_step_kernel<T, 2, 1>), grid, block, 0, stream, p);
  else if (p.dk_ <= 32)
    hipLaunchKernelGGL((delta_step_kernel<T, 4, 1>), grid, block, 0, stream, p);
  else if (p.dk_ <= 64)
    hipLaunchKernelGGL((delta_step_kernel<T, 8, 1>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((delta_step_kernel<T, 16, 1>), grid, block, 0, stream, p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_delta_step(const DeltaStepParams& p, int dtype, hipStream_t stream) {
  return dtype == 0 ? step<float>(p, stream) : step<__bf16>(p, stream);
}

}  // namespace osm
