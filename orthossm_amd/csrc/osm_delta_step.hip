// The gated delta rule token by token on gfx950: one token of a served row, or
// a short sequence.  Per state column j, with a = S^T k and b = S^T q of the
// state before the token, everything the token needs is two dot products of
// one read of the state:
//   u = beta (v - e^g a),  o = scale (e^g b + (k.q) u),  S <- e^g S + k u
//
// A workgroup holds 32 columns of a head's state in registers, its 8 row groups
// of R rows each added through two waves' shuffle and LDS: one barrier a token.
// One token is bound by the state's bytes (read and written once, 128-byte
// pieces of rows), or by the launch when there are few rows.
#include "osm_delta.h"

namespace osm {
namespace {

using namespace delta;

constexpr int kCols = 32, kGroups = 8, kStepThreads = kCols * kGroups;

template <typename T, int R>
__global__ void __launch_bounds__(kStepThreads) delta_step_kernel(const DeltaStepParams p) {
  constexpr int kRows = R * kGroups;
  __shared__ __attribute__((aligned(16))) float kq[2][2][kRows];
  __shared__ float red[2][4][3][kCols];
  const int ncb = (p.dv_ + kCols - 1) / kCols;
  const int tid = threadIdx.x, jl = tid % kCols, kg = tid / kCols, wave = tid >> 6;
  const int j = kCols * (int)(blockIdx.x % ncb) + jl, bh = blockIdx.x / ncb;
  const int b = bh / p.H, h = bh - b * p.H, hk = h / (p.H / p.Hk);
  const bool live = j < p.dv_;
  const int64_t slot = p.slots ? p.slots[b] : b;
  T* const o = row_ptr<T>(p.o, b, 0, h) + j;
  if (slot < 0 || slot >= p.n_slots) {   // an idle row, or (past the pool) a wrong one: its outputs are NaN
    if (live && kg == 0)
      for (int t = 0; t < p.S; ++t) o[t * p.o.ss] = (T)(slot < 0 ? 0.0f : __builtin_nanf(""));
    return;
  }
  const int n = p.lengths ? min(max(p.lengths[b], 0), p.S) : p.S;
  const int64_t at = slot * p.state_s + (int64_t)h * p.dk_ * p.dv_ + j;
  float s[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = kg * R + i;
    s[i] = p.init && live && row < p.dk_ ? p.init[at + (int64_t)row * p.dv_] : 0.0f;
  }
  // k and q of a token: threads 0 .. kRows-1, and the next kRows
  const bool is_q = tid >= kRows;
  const int e = is_q ? tid - kRows : tid;
  auto fetch = [&](int t) {
    if (tid >= 2 * kRows || e >= p.dk_) return 0.0f;
    return (float)(is_q ? row_ptr<T>(p.q, b, t, hk) : row_ptr<T>(p.k, b, t, hk))[e];
  };
  if (n > 0 && tid < 2 * kRows) kq[0][is_q][e] = fetch(0);
  __syncthreads();
  for (int t = 0; t < n; ++t) {
    const int par = t & 1;
    const float next = t + 1 < n ? fetch(t + 1) : 0.0f;
    const float decay = expf(*row_ptr<float>(p.g, b, t, h)), beta = *row_ptr<float>(p.beta, b, t, h);
    const float v = live ? (float)row_ptr<T>(p.v, b, t, h)[j] : 0.0f;
    float kk[R], sum[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const float q = kq[par][1][kg * R + i];
      kk[i] = kq[par][0][kg * R + i];
      sum[0] = __builtin_fmaf(s[i], kk[i], sum[0]);
      sum[1] = __builtin_fmaf(s[i], q, sum[1]);
      sum[2] = __builtin_fmaf(q, kk[i], sum[2]);
    }
#pragma unroll
    for (int c = 0; c < 3; ++c) {
      sum[c] += __shfl_xor(sum[c], 32);
      if ((tid & 32) == 0) red[par][wave][c][jl] = sum[c];
    }
    if (tid < 2 * kRows) kq[par ^ 1][is_q][e] = next;
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 3; ++c)
      sum[c] = (red[par][0][c][jl] + red[par][1][c][jl]) + (red[par][2][c][jl] + red[par][3][c][jl]);
    const float u = beta * (v - decay * sum[0]);
#pragma unroll
    for (int i = 0; i < R; ++i) s[i] = __builtin_fmaf(kk[i], u, decay * s[i]);
    if (live && kg == 0) o[t * p.o.ss] = (T)(p.scale * __builtin_fmaf(sum[2], u, decay * sum[1]));
  }
  if (live && kg == 0)
    for (int t = n; t < p.S; ++t) o[t * p.o.ss] = (T)0.0f;
  if (p.fin && live)
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int row = kg * R + i;
      if (row < p.dk_) p.fin[at + (int64_t)row * p.dv_] = s[i];
    }
}

template <typename T>
hipError_t step(const DeltaStepParams& p, hipStream_t stream) {
  const dim3 grid((unsigned)((int64_t)p.B * p.H * ((p.dv_ + kCols - 1) / kCols))), block(kStepThreads);
  if (p.dk_ <= 16)
    hipLaunchKernelGGL((delta_step_kernel<T, 2>), grid, block, 0, stream, p);
  else if (p.dk_ <= 32)
    hipLaunchKernelGGL((delta_step_kernel<T, 4>), grid, block, 0, stream, p);
  else if (p.dk_ <= 64)
    hipLaunchKernelGGL((delta_step_kernel<T, 8>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((delta_step_kernel<T, 16>), grid, block, 0, stream, p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_delta_step(const DeltaStepParams& p, int dtype, hipStream_t stream) {
  return dtype == 0 ? step<float>(p, stream) : step<__bf16>(p, stream);
}

}  // namespace osm
