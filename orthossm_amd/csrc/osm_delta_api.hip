// C ABI of the gated delta rule: argument checks, memory layout and dispatch.
// Declared in include/osm.h.
#include <algorithm>

#include "osm.h"
#include "osm_delta.h"
#include "osm_kernels.h"

namespace {

using osm::DeltaParams;
using osm::DeltaRows;
using osm::fail;
using osm::ok;

// Sequences up to this many tokens walk the state token by token in one launch
// (the step kernel) when nothing is saved for a backward.  Tokens against chunks,
// bf16, d = 64: 8 heads of 4 tokens 11.2 and 20.3 us, of 8 17.9 and 20.3, of 16 31.8
// and 20.5; 512 heads of 8 23.9 and 26.2, of 16 39.7 and 25.5.
constexpr int64_t kShort = 8;

constexpr int64_t kMaxDim = (int64_t(1) << 31) - 1;
// Workgroups of a launch: at most 512 threads each, and below 2^32 threads together.
constexpr int64_t kMaxGroups = (int64_t(1) << 23) - 1;

int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }
int64_t chunks_of(int64_t S) { return (S + osm::kDeltaChunk - 1) / osm::kDeltaChunk; }

int check_common(int32_t abi, int32_t dtype, int64_t B, int64_t H, int64_t Hk, int64_t dk, int64_t dv) {
  if (abi != OSM_ABI_VERSION) return fail(OSM_E_ARG, "abi_version %d does not match library ABI %d", abi, OSM_ABI_VERSION);
  static_assert(OSM_DELTA_MAX_DK == osm::kDeltaMaxDk, "the header states the kernels' limit");
  if (dtype != OSM_F32 && dtype != OSM_BF16) return fail(OSM_E_DTYPE, "dtype %d unsupported", dtype);
  if (B < 0) return fail(OSM_E_SHAPE, "B=%lld must be >= 0", (long long)B);
  if (H < 1 || Hk < 1 || H % Hk) return fail(OSM_E_SHAPE, "H=%lld must be a multiple of Hk=%lld", (long long)H, (long long)Hk);
  if (dk < 1 || dk > OSM_DELTA_MAX_DK) return fail(OSM_E_SHAPE, "dk=%lld outside [1, %d]", (long long)dk, OSM_DELTA_MAX_DK);
  if (dv < 1 || dv > 65536) return fail(OSM_E_SHAPE, "dv=%lld outside [1, 65536]", (long long)dv);
  if (H > 65536 || B > kMaxDim / H) return fail(OSM_E_SHAPE, "B=%lld and H=%lld too large", (long long)B, (long long)H);
  return OSM_OK;
}

// (the stride of a single token is not used: it can be anything)
int check_rows(const osm_rows& r, int esize, int64_t S, const char* name) {
  if (!r.p) return fail(OSM_E_ARG, "%s is NULL", name);
  if ((uintptr_t)r.p % esize) return fail(OSM_E_LAYOUT, "%s is not aligned to its elements", name);
  if (r.stride_b < 0 || (S > 1 && r.stride_s < 0) || r.stride_h < 0)
    return fail(OSM_E_LAYOUT, "%s has a negative stride", name);
  if (S > 1 && r.stride_s > OSM_DELTA_MAX_STRIDE)
    return fail(OSM_E_LAYOUT, "%s: %lld elements from token to token, at most %d", name, (long long)r.stride_s, OSM_DELTA_MAX_STRIDE);
  return OSM_OK;
}

// Rows of d elements over S tokens: a chunk's rows are told from those past it by
// their offset.
int check_tokens(const osm_rows& r, int esize, int64_t S, int64_t d, const char* name) {
  const int rc = check_rows(r, esize, S, name);
  if (rc == OSM_OK && S > 1 && r.stride_s < d)
    return fail(OSM_E_LAYOUT, "%s: %lld elements from token to token, rows of %lld overlap", name, (long long)r.stride_s, (long long)d);
  return rc;
}

int check_state(const void* p, const char* name) {
  return (uintptr_t)p % 4 ? fail(OSM_E_LAYOUT, "%s must be 4-byte aligned", name) : OSM_OK;
}

int check_shape(const osm_delta_args* a) {
  if (!a) return fail(OSM_E_ARG, "args is NULL");
  const int rc = check_common(a->abi_version, a->dtype, a->B, a->H, a->Hk, a->dk, a->dv);
  if (rc != OSM_OK) return rc;
  if (a->S < 0 || a->S > kMaxDim - osm::kDeltaChunk) return fail(OSM_E_SHAPE, "S=%lld outside [0, 2^31 - 64)", (long long)a->S);
  const int64_t heads = a->B * a->H, nvb = (up16(a->dv) + 63) / 64, slices = up16(a->dv) / osm::kDeltaSlice;
  const double tokens = (double)a->B * a->S * a->Hk * a->dk;   // elements of q, one a thread where heads are folded
  if (chunks_of(a->S) * nvb > kMaxGroups / std::max<int64_t>(1, heads) || slices > kMaxGroups / (heads + 7) ||
      tokens > 4294967040.0)
    return fail(OSM_E_SHAPE, "B=%lld S=%lld H=%lld Hk=%lld dk=%lld dv=%lld: too many workgroups", (long long)a->B,
                (long long)a->S, (long long)a->H, (long long)a->Hk, (long long)a->dk, (long long)a->dv);
  return OSM_OK;
}


bool is_short(const osm_delta_args* a) { return !a->saved && a->S <= kShort; }

int64_t up32(int64_t n) { return (n + 31) / 32 * 32; }

// Floats of the regions of `saved` and the workspaces, each a multiple of 64:
// per chunk Z, its gates and its start state (in the backward, the gradient to its
// end state); per segment the map and the state; with shared heads q's and k's
// gradients by head.
struct Sizes {
  size_t z, gates, s, seg_a, seg_x, part;
};
Sizes sizes_of(const osm_delta_args* a) {
  const size_t heads = (size_t)a->B * a->H, N = chunks_of(a->S), n = heads * N, dkp = up32(a->dk), dvp = up16(a->dv);
  const size_t seg = N ? osm::delta_segment(heads, N) : 1, segs = (N + seg - 1) / seg;
  const size_t m = segs > 1 ? heads * segs : 0;
  return {n * osm::kZFloats, n * osm::kGateFloats, n * dkp * dvp, m * dkp * dkp, m * dkp * dvp,
          a->H != a->Hk ? (size_t)2 * a->B * a->S * a->H * a->dk : 0};
}

DeltaRows rows_of(const osm_rows& r) { return {r.p, r.stride_b, r.stride_s, r.stride_h}; }

// Rows of d elements over S tokens as the kernels address them: a chunk's rows past
// its tokens are told by their offset, so a single token, whose stride can be
// anything, gets one that holds its row (a multiple of 4, as wide accesses want it).
osm_rows token_rows(osm_rows r, int64_t S, int64_t d) {
  if (S == 1) r.stride_s = (d + 3) / 4 * 4;
  return r;
}

bool whole(const osm_rows& r, int esize, int n) {
  return (uintptr_t)r.p % (n * esize) == 0 && r.stride_b % n == 0 && r.stride_s % n == 0 && r.stride_h % n == 0;
}

int check_inputs(const osm_delta_args* a) {
  int rc = check_shape(a);
  if (rc != OSM_OK) return rc;
  const int es = a->dtype == OSM_F32 ? 4 : 2;
  if (a->B > 0 && a->S > 0) {
    if ((rc = check_tokens(a->q, es, a->S, a->dk, "q")) != OSM_OK || (rc = check_tokens(a->k, es, a->S, a->dk, "k")) != OSM_OK ||
        (rc = check_tokens(a->v, es, a->S, a->dv, "v")) != OSM_OK || (rc = check_rows(a->g, 4, a->S, "g")) != OSM_OK ||
        (rc = check_rows(a->beta, 4, a->S, "beta")) != OSM_OK)
      return rc;
    if ((uintptr_t)a->lengths % 4) return fail(OSM_E_LAYOUT, "lengths must be 4-byte aligned");
    if ((uintptr_t)a->saved % 256) return fail(OSM_E_WORKSPACE, "saved must be 256-byte aligned");
  }
  return OSM_OK;
}

int check_workspace(const void* ws, size_t have, size_t need) {
  if (need == 0) return OSM_OK;
  if (!ws) return fail(OSM_E_WORKSPACE, "workspace is NULL");
  if ((uintptr_t)ws % 256) return fail(OSM_E_WORKSPACE, "workspace must be 256-byte aligned");
  if (have < need) return fail(OSM_E_WORKSPACE, "workspace has %zu bytes, needs %zu", have, need);
  return OSM_OK;
}

DeltaParams params_of(const osm_delta_args* a) {
  DeltaParams p{};
  const osm_rows q = token_rows(a->q, a->S, a->dk), k = token_rows(a->k, a->S, a->dk), v = token_rows(a->v, a->S, a->dv);
  p.q = rows_of(q);
  p.k = rows_of(k);
  p.v = rows_of(v);
  p.g = rows_of(a->g);
  p.beta = rows_of(a->beta);
  p.lengths = a->lengths;
  p.init = a->state_init;
  p.fin = a->state_out;
  p.B = (int)a->B;
  p.S = (int)a->S;
  p.H = (int)a->H;
  p.Hk = (int)a->Hk;
  p.dk_ = (int)a->dk;
  p.dv_ = (int)a->dv;
  p.dkp = (int)up32(a->dk);
  p.dvp = (int)up16(a->dv);
  p.N = (int)chunks_of(a->S);
  p.seg = osm::delta_segment(a->B * a->H, p.N);
  p.segs = (p.N + p.seg - 1) / p.seg;
  p.scale = a->scale;
  const int es = a->dtype == OSM_F32 ? 4 : 2;
  for (p.vec = 4; p.vec > 1; p.vec /= 2)
    if (a->dk % p.vec == 0 && a->dv % p.vec == 0 && whole(q, es, p.vec) && whole(k, es, p.vec) && whole(v, es, p.vec))
      break;
  return p;
}

// The state where a row has no tokens: dst = src, or zeros.
int copy_state(const float* src, float* dst, size_t n, hipStream_t st) {
  if (!dst || n == 0 || src == dst) return ok();
  const hipError_t e = src ? osm::launch_copy_state(src, dst, n, st) : osm::launch_fill_zero(dst, n * sizeof(float), st);
  return e == hipSuccess ? ok() : fail(OSM_E_HIP, "state copy launch: %s", hipGetErrorString(e));
}

}  // namespace

extern "C" {

size_t osm_delta_saved_bytes(const osm_delta_args* a) {
  if (check_shape(a) != OSM_OK) return 0;
  const Sizes n = sizes_of(a);
  return (n.z + n.s + n.gates) * sizeof(float);
}

size_t osm_delta_workspace_bytes(const osm_delta_args* a) {
  if (check_shape(a) != OSM_OK || is_short(a)) return 0;
  const Sizes n = sizes_of(a);
  return (n.seg_a + n.seg_x + (a->saved ? 0 : n.z + n.gates)) * sizeof(float);
}

int osm_delta_fwd(const osm_delta_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_inputs(a);
  if (rc != OSM_OK) return rc;
  if ((rc = check_state(a->state_init, "state_init")) != OSM_OK || (rc = check_state(a->state_out, "state_out")) != OSM_OK)
    return rc;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (a->B == 0 || a->S == 0) return copy_state(a->state_init, a->state_out, (size_t)a->B * a->H * a->dk * a->dv, st);
  if ((rc = check_tokens(a->out, a->dtype == OSM_F32 ? 4 : 2, a->S, a->dv, "out")) != OSM_OK) return rc;
  DeltaParams p = params_of(a);
  p.o = rows_of(token_rows(a->out, a->S, a->dv));
  hipError_t e;
  if (is_short(a)) {
    osm::DeltaStepParams s{};
    s.q = p.q;
    s.k = p.k;
    s.v = p.v;
    s.o = p.o;
    s.g = p.g;
    s.beta = p.beta;
    s.init = a->state_init;
    s.fin = a->state_out;
    s.state_s = a->H * a->dk * a->dv;
    s.n_slots = a->B;
    s.lengths = a->lengths;
    s.B = p.B;
    s.S = p.S;
    s.H = p.H;
    s.Hk = p.Hk;
    s.dk_ = p.dk_;
    s.dv_ = p.dv_;
    s.scale = p.scale;
    e = osm::launch_delta_step(s, a->dtype, st);
  } else {
    if ((rc = check_workspace(workspace, workspace_bytes, osm_delta_workspace_bytes(a))) != OSM_OK) return rc;
    const Sizes n = sizes_of(a);
    p.a = static_cast<float*>(workspace);
    p.x = p.a + n.seg_a;
    p.z = a->saved ? static_cast<float*>(a->saved) : p.x + n.seg_x;
    p.gates = p.z + n.z;
    p.s = a->saved ? p.gates + n.gates : nullptr;
    e = osm::launch_delta_fwd(p, a->dtype, st);
  }
  return e == hipSuccess ? ok() : fail(OSM_E_HIP, "delta forward launch: %s", hipGetErrorString(e));
}

size_t osm_delta_bwd_workspace_bytes(const osm_delta_args* a) {
  if (check_shape(a) != OSM_OK) return 0;
  const Sizes n = sizes_of(a);
  return (n.seg_a + n.seg_x + n.s + n.part) * sizeof(float);
}

int osm_delta_bwd(const osm_delta_args* a, const osm_delta_bwd_args* b, void* workspace, size_t workspace_bytes,
                  void* stream) {
  int rc = check_inputs(a);
  if (rc != OSM_OK) return rc;
  if (!b) return fail(OSM_E_ARG, "bwd is NULL");
  if ((rc = check_state(b->grad_state, "grad_state")) != OSM_OK || (rc = check_state(b->grad_init, "grad_init")) != OSM_OK)
    return rc;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (a->B == 0 || a->S == 0) return copy_state(b->grad_state, b->grad_init, (size_t)a->B * a->H * a->dk * a->dv, st);
  if (!a->saved) return fail(OSM_E_ARG, "saved is NULL");
  const int es = a->dtype == OSM_F32 ? 4 : 2;
  if ((rc = check_tokens(b->grad_out, es, a->S, a->dv, "grad_out")) != OSM_OK || (rc = check_tokens(b->grad_q, es, a->S, a->dk, "grad_q")) != OSM_OK ||
      (rc = check_tokens(b->grad_k, es, a->S, a->dk, "grad_k")) != OSM_OK || (rc = check_tokens(b->grad_v, es, a->S, a->dv, "grad_v")) != OSM_OK ||
      (rc = check_rows(b->grad_g, 4, a->S, "grad_g")) != OSM_OK || (rc = check_rows(b->grad_beta, 4, a->S, "grad_beta")) != OSM_OK)
    return rc;
  if ((rc = check_workspace(workspace, workspace_bytes, osm_delta_bwd_workspace_bytes(a))) != OSM_OK) return rc;
  DeltaParams p = params_of(a);
  const Sizes n = sizes_of(a);
  p.z = static_cast<float*>(a->saved);
  p.gates = p.z + n.z;
  p.s = p.gates + n.gates;
  p.a = static_cast<float*>(workspace);
  p.x = p.a + n.seg_a;
  p.d = p.x + n.seg_x;
  const osm_rows go = token_rows(b->grad_out, a->S, a->dv), gq = token_rows(b->grad_q, a->S, a->dk),
                 gk = token_rows(b->grad_k, a->S, a->dk);
  if (!whole(go, es, p.vec)) p.vec = 1;
  // (gradients by head are in the workspace, rows of dk)
  p.out_vec = a->dk % 4 == 0 && (a->H != a->Hk || (whole(gq, es, 4) && whole(gk, es, 4)));
  p.dout = rows_of(go);
  p.dq = rows_of(gq);
  p.dk = rows_of(gk);
  p.dv = rows_of(token_rows(b->grad_v, a->S, a->dv));
  p.dg = rows_of(b->grad_g);
  p.dbeta = rows_of(b->grad_beta);
  p.grad_state = b->grad_state;
  p.grad_init = b->grad_init;
  const hipError_t e = osm::launch_delta_bwd(p, p.d + n.s, a->dtype, st);
  return e == hipSuccess ? ok() : fail(OSM_E_HIP, "delta backward launch: %s", hipGetErrorString(e));
}

int osm_delta_step(const osm_delta_step_args* a, void* stream) {
  if (!a) return fail(OSM_E_ARG, "args is NULL");
  int rc = check_common(a->abi_version, a->dtype, a->B, a->H, a->Hk, a->dk, a->dv);
  if (rc != OSM_OK) return rc;
  if ((a->dv + 31) / 32 > kMaxGroups / std::max<int64_t>(1, a->B * a->H))
    return fail(OSM_E_SHAPE, "B=%lld H=%lld dv=%lld: too many workgroups", (long long)a->B, (long long)a->H, (long long)a->dv);
  if (a->n_slots < 0 || (!a->slots && a->n_slots < a->B))
    return fail(OSM_E_SHAPE, "n_slots=%lld, B=%lld rows without slots", (long long)a->n_slots, (long long)a->B);
  if (a->B == 0) return ok();
  const int es = a->dtype == OSM_F32 ? 4 : 2;
  if ((rc = check_rows(a->q, es, 1, "q")) != OSM_OK || (rc = check_rows(a->k, es, 1, "k")) != OSM_OK ||
      (rc = check_rows(a->v, es, 1, "v")) != OSM_OK || (rc = check_rows(a->out, es, 1, "out")) != OSM_OK ||
      (rc = check_rows(a->g, 4, 1, "g")) != OSM_OK || (rc = check_rows(a->beta, 4, 1, "beta")) != OSM_OK)
    return rc;
  if (!a->state && a->n_slots > 0) return fail(OSM_E_ARG, "state is NULL");
  if ((rc = check_state(a->state, "state")) != OSM_OK) return rc;
  if ((uintptr_t)a->slots % 8) return fail(OSM_E_LAYOUT, "slots must be 8-byte aligned");
  if (a->n_slots > 1 && a->state_stride < a->H * a->dk * a->dv)
    return fail(OSM_E_LAYOUT, "state_stride=%lld: slots overlap", (long long)a->state_stride);
  osm::DeltaStepParams s{};
  s.q = rows_of(a->q);
  s.k = rows_of(a->k);
  s.v = rows_of(a->v);
  s.o = rows_of(a->out);
  s.g = rows_of(a->g);
  s.beta = rows_of(a->beta);
  s.init = a->state;
  s.fin = a->state;
  s.state_s = a->state_stride;
  s.slots = a->slots;
  s.n_slots = a->n_slots;
  s.B = (int)a->B;
  s.S = 1;
  s.H = (int)a->H;
  s.Hk = (int)a->Hk;
  s.dk_ = (int)a->dk;
  s.dv_ = (int)a->dv;
  s.scale = a->scale;
  const hipError_t e = osm::launch_delta_step(s, a->dtype, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? ok() : fail(OSM_E_HIP, "delta step launch: %s", hipGetErrorString(e));
}

}  // extern "C"
