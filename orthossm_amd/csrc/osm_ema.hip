// The EMA with a learned gate on gfx950: forward, backward, one token.
//
//   h_t = a_t h_{t-1} + o_t x_t,   a = sigmoid(f),  o = 1 - a = sigmoid(-f)
//   p_t = dL/dh_t + q_t,  q_{t-1} = a_t p_t;   dx = o p,  df = a o (h_{t-1} - x) p
//
// Every token is an affine map of the state before it (the backward: of q after
// it), and maps compose.  A tile is 128 tokens of 128 channels: eight waves of
// 16 tokens, two channels a lane, whose tokens stay in registers, so every input is
// read once.  The waves' maps meet in LDS; a tile publishes its map, reads those of
// the tiles ahead of it in its group of eight and the state after the group before
// (which the group's last tile publishes), and runs its tokens from there.  The
// order of composition is fixed, so results do not depend on timing.
//
// What bounds both: the bytes of x, gate, h (x, gate, dh, dx, dgate).  8x32768x1024 bf16:
// forward 335 us, 4.8 TB/s, backward, in tiles of 64 tokens since it holds twice as much of
// each, 605 us, 4.4 TB/s (groups of four tiles: 337 and 610).  Few lane-blocks: the chain
// from group to group (bf16, 1x32768x512, 4 of them: forward 50 us, 2.0 TB/s; 1x32768x2048, 16:
// 96 us, 4.2 TB/s).
//
// The tiles that a block waits for are at work before it is: where the lane-blocks are a
// multiple of 8, blocks take their tiles by index, and those of a lane-block are on one
// XCD, to which blocks go in the order of their index; else a block draws its tile from
// its lane-block's counter when it starts (8x32768x1024 bf16, by index and drawn: 346 and
// 368 us forward, 614 and 648 backward).  The waits are bounded all the same; one that
// gives up makes NaN of what depends on it and sets the workspace's fault word.
#include <algorithm>
#include <type_traits>

#include "osm_device.h"
#include "osm_ema.h"
#include "osm_kernels.h"
#include "osm_wide_store.h"

namespace osm {
namespace {

constexpr int kThreads = kEmaWaves * 64;
constexpr float kTiny = 1.17549435e-38f;   // the least normal number

typedef float F2 __attribute__((ext_vector_type(2)));

// Two channels of a row as loaded.
template <typename T>
struct Pair {
  typedef T V __attribute__((ext_vector_type(2)));
  V v;
};

template <typename T, bool VEC>
__device__ __forceinline__ Pair<T> load_pair(const T* p, int c, int D) {
  Pair<T> r;
  if constexpr (VEC) {
    r.v = __builtin_nontemporal_load(reinterpret_cast<const typename Pair<T>::V*>(p + c));
  } else {
    r.v.x = p[c];
    r.v.y = c + 1 < D ? p[c + 1] : (T)0.0f;
  }
  return r;
}

template <typename T, bool VEC>
__device__ __forceinline__ void store_pair(T* p, int c, int D, F2 v) {
  const typename Pair<T>::V q = {(T)v.x, (T)v.y};
  if constexpr (VEC) {
    __builtin_nontemporal_store(q, reinterpret_cast<typename Pair<T>::V*>(p + c));
  } else {
    p[c] = q.x;
    if (c + 1 < D) p[c + 1] = q.y;
  }
}

// sigmoid(f) and sigmoid(-f), off by |f| 2^-24 and a few units of 2^-24.
struct Sig {
  float a, o;
};
__device__ __forceinline__ Sig sigmoids(float f) {
  const float e = __builtin_amdgcn_exp2f(-1.44269504f * __builtin_fabsf(f));
  // the smaller of the two by the reciprocal, the larger as what it leaves of 1: they
  // add up to 1, and a decay next to 1 is rounded once (its error counts as often as
  // the state remembers)
  const float s = e * __builtin_amdgcn_rcpf(1.0f + e), r = 1.0f - s;
  Sig g;
  g.a = f >= 0.0f ? r : s;
  g.o = f >= 0.0f ? s : r;
  return g;
}
struct Sig2 {
  F2 a, o;
};
template <typename T>
__device__ __forceinline__ Sig2 sigmoids(const Pair<T>& f) {
  const Sig u = sigmoids((float)f.v.x), v = sigmoids((float)f.v.y);
  return {{u.a, v.a}, {u.o, v.o}};
}

__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  return F2{__builtin_fmaf(a.x, b.x, c.x), __builtin_fmaf(a.y, b.y, c.y)};
}
// A composed decay does not underflow to 0: an infinite state stays infinite, and a
// published map is never the word 0.
__device__ __forceinline__ F2 floor2(F2 a) { return F2{__builtin_fmaxf(a.x, kTiny), __builtin_fmaxf(a.y, kTiny)}; }

__device__ __forceinline__ F2 state2(const float* p, int64_t at, int c, int D) {
  if (!p) return F2{0.0f, 0.0f};
  return F2{p[at + c], c + 1 < D ? p[at + c + 1] : 0.0f};
}
// (rows of an even D are whole pairs)
__device__ __forceinline__ void put_saved(float* p, int64_t at, int c, int D, F2 v) {
  if (D % 2 == 0) {
    *reinterpret_cast<F2*>(p + at + c) = v;
  } else {
    p[at + c] = v.x;
    if (c + 1 < D) p[at + c + 1] = v.y;
  }
}
__device__ __forceinline__ void put2(float* p, int64_t at, int c, int D, F2 v) {
  p[at + c] = v.x;
  if (c + 1 < D) p[at + c + 1] = v.y;
}

// Until these are in registers.  (A state may lie where another block writes the one it
// hands on: that block waits for what is posted after this.)
__device__ __forceinline__ void arrive(F2 v) { asm volatile("" ::"v"(v.x), "v"(v.y)); }

// Waits for a word to be published (they are never 0): its producer has been running
// since before this block drew its tile.  A wait that gives up sets the fault word.
__device__ __forceinline__ unsigned long long await(const unsigned long long* at, const EmaParams& p) {
  unsigned long long w = peek(at);
  for (unsigned polls = 0; w == 0 && polls < p.poll_limit; ++polls) {
    __builtin_amdgcn_s_sleep(1);
    w = peek(at);
  }
  if (w) return w;
  raise_fault(p.lines, kKindFault);
  return 0x7fc000007fc00000ull;   // NaN, NaN
}
__device__ __forceinline__ unsigned long long word_of(float hi, float lo) {
  return (unsigned long long)__float_as_uint(hi) << 32 | __float_as_uint(lo);
}
__device__ __forceinline__ void post(unsigned long long* at, float hi, float lo) {
  __hip_atomic_store(at, word_of(hi, lo), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

struct Shared {
  F2 a[kEmaWaves][64], b[kEmaWaves][64];   // the waves' maps
  F2 pa[kEmaGroup][64], pb[kEmaGroup][64];   // the maps of tiles ahead; [kEmaGroup - 1]: pb holds the state after the group before
  int drawn;
};

struct Place {
  int lane, wave, lb, b, c, tile;
};

// This block's place.
__device__ __forceinline__ Place place(const EmaParams& p, Shared& L) {
  Place q;
  q.lane = threadIdx.x & 63;
  q.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  q.lb = blockIdx.x % p.n_lb;
  q.b = q.lb / p.n_lbd;
  q.c = (q.lb - q.b * p.n_lbd) * kEmaLanes + 2 * q.lane;
  q.tile = 0;
  if (p.n_lb % 8 == 0) {
    q.tile = blockIdx.x / p.n_lb;
  } else if (p.n_tiles > 1) {
    if (threadIdx.x == 0)
      L.drawn = (int)__hip_atomic_fetch_add(p.lines + (int64_t)q.lb * kEmaLine + kEmaTicket, 1u, __ATOMIC_RELAXED,
                                            __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    q.tile = __builtin_amdgcn_readfirstlane(L.drawn);
  }
  return q;
}

__device__ __forceinline__ int tokens_of(const EmaParams& p, int b) {
  return p.lengths ? min(max(p.lengths[b], 0), p.S) : p.S;
}

// The carry into tile j of a lane-block's chain, where the waves' maps lie in L.a
// and L.b (in the chain's order where `back` is false, else reversed) and the chain
// starts from `start`.  Posts this tile's map, or the state after its group.
__device__ __forceinline__ F2 carry_in(const EmaParams& p, Shared& L, const Place& q, int j, bool last, bool back, F2 start) {
  const int k = j % kEmaGroup, g = j / kEmaGroup;
  F2 A = {1.0f, 1.0f}, B = {0.0f, 0.0f};
  if (q.wave == 0 && !last) {
#pragma unroll
    for (int i = 0; i < kEmaWaves; ++i) {
      const int w = back ? kEmaWaves - 1 - i : i;
      B = fma2(L.a[w][q.lane], B, L.b[w][q.lane]);
      A = floor2(A * L.a[w][q.lane]);
    }
    if (k != kEmaGroup - 1) {
      unsigned long long* const w = p.words + ((int64_t)q.lb * p.n_tiles + j) * kEmaLanes + 2 * q.lane;
      post(w, A.x, B.x);
      post(w + 1, A.y, B.y);
    }
  }
  if (j > 0) {
    if (q.wave < k) {
      const unsigned long long* const w = p.words + ((int64_t)q.lb * p.n_tiles + g * kEmaGroup + q.wave) * kEmaLanes + 2 * q.lane;
      const unsigned long long u = await(w, p), v = await(w + 1, p);
      L.pa[q.wave][q.lane] = F2{__uint_as_float((unsigned)(u >> 32)), __uint_as_float((unsigned)(v >> 32))};
      L.pb[q.wave][q.lane] = F2{__uint_as_float((unsigned)u), __uint_as_float((unsigned)v)};
    } else if (q.wave == kEmaGroup - 1 && g > 0) {
      const unsigned long long* const w = p.marks + ((int64_t)q.lb * p.n_groups + g - 1) * kEmaLanes + 2 * q.lane;
      const unsigned long long u = await(w, p), v = await(w + 1, p);
      L.pb[kEmaGroup - 1][q.lane] = F2{__uint_as_float((unsigned)u), __uint_as_float((unsigned)v)};
    }
    __syncthreads();
    if (g > 0) start = L.pb[kEmaGroup - 1][q.lane];
    for (int i = 0; i < k; ++i) start = fma2(L.pa[i][q.lane], start, L.pb[i][q.lane]);
  }
  if (q.wave == 0 && !last && k == kEmaGroup - 1) {
    const F2 s = fma2(A, start, B);
    unsigned long long* const w = p.marks + ((int64_t)q.lb * p.n_groups + g) * kEmaLanes + 2 * q.lane;
    post(w, 1.0f, s.x);
    post(w + 1, 1.0f, s.y);
  }
  return start;
}

// A wave's tokens of a sequence: token t0 + i at each step of i.
template <typename T>
__device__ __forceinline__ T* first_row(const EmaSeq& s, const Place& q, int64_t t) {
  return static_cast<T*>(s.p) + q.b * s.sb + t * s.ss;
}
template <typename T, bool VEC, int R>
__device__ __forceinline__ void load_run(Pair<T> (&v)[R], const EmaSeq& s, const Place& q, int t0, int len, int c, int D) {
  const T* row = first_row<T>(s, q, min(t0, len - 1));   // (rows past the last token: that one again)
#pragma unroll
  for (int i = 0; i < R; ++i) {
    v[i] = load_pair<T, VEC>(row, c, D);
    row += t0 + i + 1 < len ? s.ss : 0;
  }
}

// Tokens past the last of a run, as if their gate were open for good: h and q go through.
template <typename T, int R>
__device__ __forceinline__ void blank(Pair<T> (&v)[R], int n, float with) {
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (i >= n) v[i].v = {(T)with, (T)with};
}

// Zeros of a tile past its row's tokens.
template <typename T, bool VEC, int R>
__device__ __forceinline__ void zero_tile(const EmaParams& p, const EmaSeq& s, const Place& q) {
  const int t0 = (q.tile * kEmaWaves + q.wave) * R;
  T* row = first_row<T>(s, q, t0);
  for (int i = 0; i < R && t0 + i < p.S; ++i, row += s.ss) store_pair<T, VEC>(row, q.c, p.D, F2{0.0f, 0.0f});
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads, 4) ema_fwd_kernel(const EmaParams p) {
  constexpr int R = kEmaRun, kTile = kEmaTile;
  __shared__ Shared L;
  const Place q = place(p, L);
  const int len = tokens_of(p, q.b), D = p.D;
  const bool live = q.c < D;
  if (q.tile * kTile >= len) {   // (nothing waits for this tile)
    if (!live) return;
    if (q.tile == 0 && q.wave == 0 && p.fin) put2(p.fin, (int64_t)q.b * D, q.c, D, state2(p.init, (int64_t)q.b * D, q.c, D));
    zero_tile<T, VEC, R>(p, p.out, q);
    return;
  }
  const int t0 = q.tile * kTile + q.wave * R, n = len - t0;   // n: tokens from t0 on
  Pair<T> rx[R], rf[R];
  const int c = live ? q.c : 0;
  load_run<T, VEC>(rf, p.gate, q, t0, len, c, D);
  load_run<T, VEC>(rx, p.x, q, t0, len, c, D);
  const F2 start = live ? state2(p.init, (int64_t)q.b * D, q.c, D) : F2{0.0f, 0.0f};
  if (n < R) {
    blank(rf, n, __builtin_inff());
    blank(rx, n, 0.0f);
  }
  F2 a[R], b[R], A = {1.0f, 1.0f}, B = {0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const Sig2 s = sigmoids(rf[i]);
    a[i] = s.a;
    b[i] = s.o * F2{(float)rx[i].v.x, (float)rx[i].v.y};
    A = A * a[i];
    B = fma2(a[i], B, b[i]);
  }
  L.a[q.wave][q.lane] = floor2(A);
  L.b[q.wave][q.lane] = B;
  arrive(start);
  __syncthreads();
  F2 h = carry_in(p, L, q, q.tile, (q.tile + 1) * kTile >= len, false, start);
  if (!live) return;
  for (int w = 0; w < q.wave; ++w) h = fma2(L.a[w][q.lane], h, L.b[w][q.lane]);
  if (p.saved && n > 0 && t0 % kEmaBwdTile == 0)
    put_saved(p.saved, ((int64_t)q.b * p.n_saved + t0 / kEmaBwdTile) * D, q.c, D, h);
  T* row = first_row<T>(p.out, q, t0);
  if (n >= R) {
#pragma unroll
    for (int i = 0; i < R; ++i, row += p.out.ss) {
      h = fma2(a[i], h, b[i]);
      store_pair<T, VEC>(row, q.c, D, h);
    }
  } else {
#pragma unroll
    for (int i = 0; i < R; ++i, row += p.out.ss) {
      h = fma2(a[i], h, b[i]);
      if (t0 + i < p.S) store_pair<T, VEC>(row, q.c, D, i < n ? h : F2{0.0f, 0.0f});
    }
  }
  if (p.fin && n > 0 && n <= R) put2(p.fin, (int64_t)q.b * D, q.c, D, h);
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads, 4) ema_bwd_kernel(const EmaParams p) {
  constexpr int R = kEmaBwdRun, kTile = kEmaBwdTile;
  __shared__ Shared L;
  __shared__ F2 fb[kEmaWaves][64];   // the waves' maps of h (L.b: of q; the factors are the same)
  Place q = place(p, L);
  q.tile = p.n_tiles - 1 - q.tile;
  const int len = tokens_of(p, q.b), D = p.D;
  const bool live = q.c < D;
  if (q.tile * kTile >= len) {
    if (!live) return;
    if (q.tile == 0 && q.wave == 0 && p.ginit)
      put2(p.ginit, (int64_t)q.b * D, q.c, D, state2(p.gstate, (int64_t)q.b * D, q.c, D));
    zero_tile<T, VEC, R>(p, p.gx, q);
    zero_tile<T, VEC, R>(p, p.gg, q);
    return;
  }
  const int t0 = q.tile * kTile + q.wave * R, n = len - t0;
  Pair<T> rx[R], rf[R], rg[R];
  const int c = live ? q.c : 0;
  load_run<T, VEC>(rf, p.gate, q, t0, len, c, D);
  load_run<T, VEC>(rx, p.x, q, t0, len, c, D);
  load_run<T, VEC>(rg, p.go, q, t0, len, c, D);
  const F2 start = live ? state2(p.gstate, (int64_t)q.b * D, q.c, D) : F2{0.0f, 0.0f};
  F2 h = live ? state2(p.saved, ((int64_t)q.b * p.n_saved + q.tile) * D, q.c, D) : F2{0.0f, 0.0f};
  if (n < R) {
    blank(rf, n, __builtin_inff());
    blank(rx, n, 0.0f);
    blank(rg, n, 0.0f);
  }
  F2 a[R], o[R], A = {1.0f, 1.0f}, B = {0.0f, 0.0f}, Q = {0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const Sig2 s = sigmoids(rf[i]);
    a[i] = s.a;
    o[i] = s.o;
    A = A * a[i];
    Q = fma2(A, F2{(float)rg[i].v.x, (float)rg[i].v.y}, Q);   // (q ahead of the run, of none after it)
    B = fma2(a[i], B, o[i] * F2{(float)rx[i].v.x, (float)rx[i].v.y});
  }
  L.a[q.wave][q.lane] = floor2(A);
  L.b[q.wave][q.lane] = Q;
  fb[q.wave][q.lane] = B;
  arrive(start);
  __syncthreads();
  const int used = (len + kTile - 1) / kTile;
  F2 g = carry_in(p, L, q, used - 1 - q.tile, q.tile == 0, true, start);
  if (!live) return;
  for (int w = 0; w < q.wave; ++w) h = fma2(L.a[w][q.lane], h, fb[w][q.lane]);
  for (int w = kEmaWaves - 1; w > q.wave; --w) g = fma2(L.a[w][q.lane], g, L.b[w][q.lane]);
  F2 d[R];   // a (h_{t-1} - x_t)
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const F2 x = {(float)rx[i].v.x, (float)rx[i].v.y};
    d[i] = a[i] * (h - x);
    h = fma2(a[i], h, o[i] * x);
  }
  T* gx = first_row<T>(p.gx, q, t0 + R);
  T* gg = first_row<T>(p.gg, q, t0 + R);
#pragma unroll
  for (int i = R - 1; i >= 0; --i) {
    gx -= p.gx.ss;
    gg -= p.gg.ss;
    const F2 u = g + F2{(float)rg[i].v.x, (float)rg[i].v.y};
    const F2 ou = o[i] * u;   // (0 past the last token: its o is)
    g = a[i] * u;
    if (n < R && t0 + i >= p.S) continue;
    store_pair<T, VEC>(gx, q.c, D, i < n ? ou : F2{0.0f, 0.0f});
    store_pair<T, VEC>(gg, q.c, D, i < n ? d[i] * ou : F2{0.0f, 0.0f});
  }
  if (p.ginit && t0 == 0) put2(p.ginit, (int64_t)q.b * D, q.c, D, g);
}

// One token a row: NC channels a thread.
template <typename T, int NC>
__global__ void __launch_bounds__(256) ema_step_kernel(const EmaStepParams p) {
  const int per = (p.D + NC - 1) / NC;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)p.B * per) return;
  const int b = (int)(i / per), c = (int)(i - (int64_t)b * per) * NC;
  const int64_t slot = p.slots ? p.slots[b] : b;
  float x[NC], f[NC], h[NC];
  T* const out = static_cast<T*>(p.out.p) + b * p.out.sb + c;
  if (slot < 0 || slot >= p.n_slots) {   // an idle row, or (past the pool) a wrong one: its outputs are NaN
#pragma unroll
    for (int k = 0; k < NC; ++k) h[k] = slot < 0 ? 0.0f : __builtin_nanf("");
    LaneVec<T, NC>::store(out, h);
    wide_store_wait();
    return;
  }
  float* const s = p.state + slot * p.state_s + c;
  LaneVec<T, NC>::load(static_cast<const T*>(p.x.p) + b * p.x.sb + c, x);
  LaneVec<T, NC>::load(static_cast<const T*>(p.gate.p) + b * p.gate.sb + c, f);
  LaneVec<float, NC>::load(s, h);
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    const Sig g = sigmoids(f[k]);
    h[k] = __builtin_fmaf(g.a, h[k], g.o * x[k]);
  }
  LaneVec<float, NC>::store(s, h);
  wide_store_wait();
  LaneVec<T, NC>::store(out, h);
  wide_store_wait();
}

// f(T{}, VEC): the kernels' version by type and alignment.
template <typename F>
hipError_t by_form(int dtype, int vec, F f) {
  auto typed = [&](auto t) {
    if (vec)
      f(t, std::true_type{});
    else
      f(t, std::false_type{});
  };
  if (dtype == 0)
    typed(0.0f);
  else
    typed((__bf16)0.0f);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_ema_fwd(const EmaParams& p, int dtype, hipStream_t stream) {
  return by_form(dtype, p.vec, [&](auto t, auto vec) {
    hipLaunchKernelGGL((ema_fwd_kernel<decltype(t), decltype(vec)::value>), dim3((unsigned)(p.n_lb * p.n_tiles)), dim3(kThreads),
                       0, stream, p);
  });
}

hipError_t launch_ema_bwd(const EmaParams& p, int dtype, hipStream_t stream) {
  return by_form(dtype, p.vec, [&](auto t, auto vec) {
    hipLaunchKernelGGL((ema_bwd_kernel<decltype(t), decltype(vec)::value>), dim3((unsigned)(p.n_lb * p.n_tiles)), dim3(kThreads),
                       0, stream, p);
  });
}

hipError_t launch_ema_step(const EmaStepParams& p, int dtype, hipStream_t stream) {
  const int64_t n = (int64_t)p.B * (p.vec ? p.D / 4 : p.D);
  return by_form(dtype, p.vec, [&](auto t, auto vec) {
    hipLaunchKernelGGL((ema_step_kernel<decltype(t), decltype(vec)::value ? 4 : 1>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0,
                       stream, p);
  });
}

}  // namespace osm
