// C ABI of the gated EMA: argument checks, memory layout and dispatch.  Declared in
// include/osm.h.
#include <algorithm>

#include "osm.h"
#include "osm_ema.h"
#include "osm_kernels.h"

namespace {

using osm::EmaParams;
using osm::EmaSeq;
using osm::fail;
using osm::kEmaGroup;
using osm::kEmaLanes;
using osm::kEmaBwdTile;
using osm::kEmaTile;
using osm::ok;

constexpr int64_t kMaxDim = (int64_t(1) << 31) - 1;
// Workgroups of a launch: 512 threads each, and below 2^32 threads together.
constexpr int64_t kMaxGroups = (int64_t(1) << 23) - 1;

int64_t div_up(int64_t n, int64_t d) { return (n + d - 1) / d; }

int check_common(int32_t abi, int32_t dtype, int64_t B, int64_t D) {
  if (abi != OSM_ABI_VERSION) return fail(OSM_E_ARG, "abi_version %d does not match library ABI %d", abi, OSM_ABI_VERSION);
  if (dtype != OSM_F32 && dtype != OSM_BF16) return fail(OSM_E_DTYPE, "dtype %d unsupported", dtype);
  if (B < 0 || D < 1 || B > kMaxDim || D > kMaxDim)
    return fail(OSM_E_SHAPE, "B=%lld must be >= 0, D=%lld >= 1, both below 2^31", (long long)B, (long long)D);
  return OSM_OK;
}

int check_seq(const osm_seq& r, int esize, int64_t S, const char* name) {
  if (!r.p) return fail(OSM_E_ARG, "%s is NULL", name);
  if ((uintptr_t)r.p % esize) return fail(OSM_E_LAYOUT, "%s is not aligned to its elements", name);
  if (r.stride_b < 0 || (S > 1 && r.stride_s < 0)) return fail(OSM_E_LAYOUT, "%s has a negative stride", name);
  return OSM_OK;
}

// An output: no element twice.
int check_out(const osm_seq& r, int esize, int64_t B, int64_t S, int64_t D, const char* name) {
  const int rc = check_seq(r, esize, S, name);
  if (rc != OSM_OK) return rc;
  // rows follow each other by token within a batch row, or by batch row within a token
  const bool by_row = (S == 1 || r.stride_s >= D) && (B == 1 || r.stride_b >= (S > 1 ? (S - 1) * r.stride_s : 0) + D);
  const bool by_token = (B == 1 || r.stride_b >= D) && (S == 1 || r.stride_s >= (B > 1 ? (B - 1) * r.stride_b : 0) + D);
  return by_row || by_token ? OSM_OK : fail(OSM_E_LAYOUT, "%s: rows overlap", name);
}

// (a test aid's bit may be beside the type)
int32_t type_of(const osm_ema_args* a) { return a->dtype & ~OSM_FLAG_POLL_LIMIT_ZERO; }
int esize_of(const osm_ema_args* a) { return type_of(a) == OSM_F32 ? 4 : 2; }

int check_shape(const osm_ema_args* a) {
  if (!a) return fail(OSM_E_ARG, "args is NULL");
  const int rc = check_common(a->abi_version, type_of(a), a->B, a->D);
  if (rc != OSM_OK) return rc;
  if (a->S < 0 || a->S > kMaxDim - 255) return fail(OSM_E_SHAPE, "S=%lld outside [0, 2^31 - 256)", (long long)a->S);
  const int64_t lbd = div_up(a->D, kEmaLanes);
  if (lbd > kMaxGroups / std::max<int64_t>(1, a->B) || div_up(a->S, kEmaBwdTile) > kMaxGroups / std::max<int64_t>(1, a->B * lbd))
    return fail(OSM_E_SHAPE, "B=%lld S=%lld D=%lld: too many workgroups", (long long)a->B, (long long)a->S, (long long)a->D);
  return OSM_OK;
}

int check_inputs(const osm_ema_args* a) {
  int rc = check_shape(a);
  if (rc != OSM_OK) return rc;
  const int es = esize_of(a);
  if (a->B > 0 && a->S > 0 &&
      ((rc = check_seq(a->x, es, a->S, "x")) != OSM_OK || (rc = check_seq(a->gate, es, a->S, "gate")) != OSM_OK))
    return rc;
  const void* words[3] = {a->lengths, a->state_init, a->state_out};
  for (const void* w : words)
    if ((uintptr_t)w % 4) return fail(OSM_E_LAYOUT, "lengths and states must be 4-byte aligned");
  if ((uintptr_t)a->saved % 256) return fail(OSM_E_LAYOUT, "saved must be 256-byte aligned");
  return OSM_OK;
}

struct Sizes {
  size_t lines, words, marks;   // bytes, in this order, zeroed ahead of a launch; 0: one tile a row
  size_t total() const { return lines + words + marks; }
};
Sizes sizes_of(const osm_ema_args* a, int tile) {
  const size_t lb = (size_t)a->B * div_up(a->D, kEmaLanes), tiles = div_up(a->S, tile);
  if (tiles <= 1 || lb == 0) return {0, 0, 0};
  return {lb * osm::kEmaLine * 4, lb * tiles * kEmaLanes * 8, lb * div_up(tiles, kEmaGroup) * kEmaLanes * 8};
}

// (the stride of a single token is not used: it can be anything)
EmaSeq seq_of(const osm_seq& r, int64_t S) { return {r.p, r.stride_b, S > 1 ? r.stride_s : 0}; }

bool pairs(const osm_seq& r, int64_t S, int esize) {
  return (uintptr_t)r.p % (2 * esize) == 0 && r.stride_b % 2 == 0 && (S == 1 || r.stride_s % 2 == 0);
}

EmaParams params_of(const osm_ema_args* a, int tile, void* workspace) {
  EmaParams p{};
  p.x = seq_of(a->x, a->S);
  p.gate = seq_of(a->gate, a->S);
  p.lengths = a->lengths;
  p.init = a->state_init;
  p.saved = a->saved;
  p.B = (int)a->B;
  p.S = (int)a->S;
  p.D = (int)a->D;
  p.n_lbd = (int)div_up(a->D, kEmaLanes);
  p.n_lb = p.B * p.n_lbd;
  p.n_tiles = (int)div_up(a->S, tile);
  p.n_saved = (int)div_up(a->S, kEmaBwdTile);
  p.n_groups = (int)div_up(p.n_tiles, kEmaGroup);
  const Sizes n = sizes_of(a, tile);
  char* const w = static_cast<char*>(workspace);
  p.lines = reinterpret_cast<unsigned*>(w);
  p.words = reinterpret_cast<unsigned long long*>(w + n.lines);
  p.marks = reinterpret_cast<unsigned long long*>(w + n.lines + n.words);
  p.poll_limit = (a->dtype & OSM_FLAG_POLL_LIMIT_ZERO) ? 0u : osm::kSpinLimit;
  const int es = esize_of(a);
  p.vec = a->D % 2 == 0 && pairs(a->x, a->S, es) && pairs(a->gate, a->S, es);
  return p;
}

int prepare(const osm_ema_args* a, int tile, void* workspace, size_t bytes, hipStream_t st) {
  const size_t need = sizes_of(a, tile).total();
  if (need == 0) return OSM_OK;
  if (!workspace || (uintptr_t)workspace % 256 || bytes < need)
    return fail(OSM_E_WORKSPACE, "the workspace must be 256-byte aligned and have %zu bytes (it has %zu)", need, workspace ? bytes : 0);
  const hipError_t e = osm::launch_fill_zero(workspace, need, st);
  return e == hipSuccess ? OSM_OK : fail(OSM_E_HIP, "workspace fill launch: %s", hipGetErrorString(e));
}

// No tokens: the state (or its gradient) goes through.
int pass_state(const osm_ema_args* a, const float* from, float* to, hipStream_t st) {
  if (!to || to == from || a->B == 0) return ok();
  const size_t n = (size_t)a->B * a->D;
  const hipError_t e = from ? osm::launch_copy_state(from, to, n, st) : osm::launch_fill_zero(to, n * sizeof(float), st);
  return e == hipSuccess ? ok() : fail(OSM_E_HIP, "state copy launch: %s", hipGetErrorString(e));
}

}  // namespace

extern "C" {

size_t osm_gated_ema_saved_bytes(const osm_ema_args* a) {
  return check_shape(a) == OSM_OK ? (size_t)a->B * div_up(a->S, kEmaBwdTile) * a->D * sizeof(float) : 0;
}

size_t osm_gated_ema_workspace_bytes(const osm_ema_args* a) {
  return check_shape(a) == OSM_OK ? sizes_of(a, kEmaTile).total() : 0;
}

size_t osm_gated_ema_bwd_workspace_bytes(const osm_ema_args* a) {
  return check_shape(a) == OSM_OK ? sizes_of(a, kEmaBwdTile).total() : 0;
}

int osm_gated_ema_fwd(const osm_ema_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_inputs(a);
  if (rc != OSM_OK) return rc;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (a->B == 0 || a->S == 0) return pass_state(a, a->state_init, a->state_out, st);
  const int es = esize_of(a);
  if ((rc = check_out(a->out, es, a->B, a->S, a->D, "out")) != OSM_OK) return rc;
  if ((rc = prepare(a, kEmaTile, workspace, workspace_bytes, st)) != OSM_OK) return rc;
  EmaParams p = params_of(a, kEmaTile, workspace);
  p.out = seq_of(a->out, a->S);
  p.fin = a->state_out;
  p.vec = p.vec && pairs(a->out, a->S, es);
  const hipError_t e = osm::launch_ema_fwd(p, type_of(a), st);
  return e == hipSuccess ? ok() : fail(OSM_E_HIP, "gated EMA launch: %s", hipGetErrorString(e));
}

int osm_gated_ema_bwd(const osm_ema_args* a, const osm_ema_bwd_args* b, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_inputs(a);
  if (rc != OSM_OK) return rc;
  if (!b) return fail(OSM_E_ARG, "bwd is NULL");
  if ((uintptr_t)b->grad_state % 4 || (uintptr_t)b->grad_init % 4)
    return fail(OSM_E_LAYOUT, "grad_state and grad_init must be 4-byte aligned");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (a->B == 0 || a->S == 0) return pass_state(a, b->grad_state, b->grad_init, st);
  if (!a->saved) return fail(OSM_E_ARG, "saved is NULL");
  const int es = esize_of(a);
  if ((rc = check_seq(b->grad_out, es, a->S, "grad_out")) != OSM_OK ||
      (rc = check_out(b->grad_x, es, a->B, a->S, a->D, "grad_x")) != OSM_OK ||
      (rc = check_out(b->grad_gate, es, a->B, a->S, a->D, "grad_gate")) != OSM_OK)
    return rc;
  if ((rc = prepare(a, kEmaBwdTile, workspace, workspace_bytes, st)) != OSM_OK) return rc;
  EmaParams p = params_of(a, kEmaBwdTile, workspace);
  p.go = seq_of(b->grad_out, a->S);
  p.gx = seq_of(b->grad_x, a->S);
  p.gg = seq_of(b->grad_gate, a->S);
  p.gstate = b->grad_state;
  p.ginit = b->grad_init;
  p.vec = p.vec && pairs(b->grad_out, a->S, es) && pairs(b->grad_x, a->S, es) && pairs(b->grad_gate, a->S, es);
  const hipError_t e = osm::launch_ema_bwd(p, type_of(a), st);
  return e == hipSuccess ? ok() : fail(OSM_E_HIP, "gated EMA backward launch: %s", hipGetErrorString(e));
}

int osm_gated_ema_step(const osm_ema_step_args* a, void* stream) {
  if (!a) return fail(OSM_E_ARG, "args is NULL");
  int rc = check_common(a->abi_version, a->dtype, a->B, a->D);
  if (rc != OSM_OK) return rc;
  if ((double)a->B * a->D > 4294967040.0)   // (threads of the launch)
    return fail(OSM_E_SHAPE, "B=%lld D=%lld: too many workgroups", (long long)a->B, (long long)a->D);
  if (a->n_slots < 0 || (!a->slots && a->n_slots < a->B))
    return fail(OSM_E_SHAPE, "n_slots=%lld, B=%lld rows without slots", (long long)a->n_slots, (long long)a->B);
  if (a->B == 0) return ok();
  const int es = a->dtype == OSM_F32 ? 4 : 2;
  if ((rc = check_seq(a->x, es, 1, "x")) != OSM_OK || (rc = check_seq(a->gate, es, 1, "gate")) != OSM_OK ||
      (rc = check_out(a->out, es, a->B, 1, a->D, "out")) != OSM_OK)
    return rc;
  if (!a->state && a->n_slots > 0) return fail(OSM_E_ARG, "state is NULL");
  if ((uintptr_t)a->state % 4) return fail(OSM_E_LAYOUT, "state must be 4-byte aligned");
  if ((uintptr_t)a->slots % 8) return fail(OSM_E_LAYOUT, "slots must be 8-byte aligned");
  if (a->n_slots > 1 && a->state_stride < a->D) return fail(OSM_E_LAYOUT, "state_stride=%lld: slots overlap", (long long)a->state_stride);
  osm::EmaStepParams p{};
  p.x = seq_of(a->x, 1);
  p.gate = seq_of(a->gate, 1);
  p.out = seq_of(a->out, 1);
  p.state = a->state;
  p.state_s = a->state_stride;
  p.n_slots = a->n_slots;
  p.slots = a->slots;
  p.B = (int)a->B;
  p.D = (int)a->D;
  auto whole = [&](const osm_seq& r) { return (uintptr_t)r.p % (4 * es) == 0 && r.stride_b % 4 == 0; };
  p.vec = a->D % 4 == 0 && whole(a->x) && whole(a->gate) && whole(a->out) && (uintptr_t)a->state % 16 == 0 && a->state_stride % 4 == 0;
  const hipError_t e = osm::launch_ema_step(p, a->dtype, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? ok() : fail(OSM_E_HIP, "gated EMA step launch: %s", hipGetErrorString(e));
}

}  // extern "C"
