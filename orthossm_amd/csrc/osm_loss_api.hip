// C ABI of the vocabulary's cross entropy: argument checks, memory layout and
// dispatch.  Declared in include/osm.h.
#include <algorithm>

#include "osm.h"
#include "osm_kernels.h"
#include "osm_loss.h"

namespace {

using osm::fail;
using osm::kLossPad;
using osm::LossParams;
using osm::ok;

constexpr int64_t kMaxRow = int64_t(1) << 21;   // elements of an operand's row

int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

int check_args(const osm_loss_args* a) {
  if (!a) return fail(OSM_E_ARG, "args is NULL");
  if (a->abi_version != OSM_ABI_VERSION)
    return fail(OSM_E_ARG, "abi_version %d does not match library ABI %d", a->abi_version, OSM_ABI_VERSION);
  if (a->flags & ~OSM_LOSS_MEAN) return fail(OSM_E_ARG, "unknown flag bits 0x%x", a->flags);
  if (a->dtype != OSM_F32 && a->dtype != OSM_BF16) return fail(OSM_E_DTYPE, "dtype %d unsupported", a->dtype);
  if (a->N < 0 || a->N > kMaxRow - kLossPad || a->D < 1 || a->D > (int64_t(1) << 17) || a->V < 1 || a->V > (int64_t(1) << 28))
    return fail(OSM_E_SHAPE, "N=%lld outside [0, 2^21 - 256], D=%lld outside [1, 2^17] or V=%lld outside [1, 2^28]", (long long)a->N,
                (long long)a->D, (long long)a->V);
  return OSM_OK;
}

int check_matrix(const void* p, int64_t stride, int64_t least, int esize, const char* name) {
  if (!p) return fail(OSM_E_ARG, "%s is NULL", name);
  if ((uintptr_t)p % esize) return fail(OSM_E_LAYOUT, "%s is not aligned to its elements", name);
  if (stride < least) return fail(OSM_E_LAYOUT, "%s: row stride %lld below %lld", name, (long long)stride, (long long)least);
  return OSM_OK;
}

int check_inputs(const osm_loss_args* a) {
  const int es = a->dtype == OSM_F32 ? 4 : 2;
  int rc;
  if ((rc = check_matrix(a->hidden, a->hidden_stride, 0, es, "hidden")) != OSM_OK ||
      (rc = check_matrix(a->weight, a->weight_stride, 0, es, "weight")) != OSM_OK)
    return rc;
  if (!a->targets || (uintptr_t)a->targets % 8) return fail(OSM_E_ARG, "targets is NULL or not 8-byte aligned");
  if (!a->lse || (uintptr_t)a->lse % 4) return fail(OSM_E_ARG, "lse is NULL or not 4-byte aligned");
  return OSM_OK;
}

// Whether the weights are read where they are.
bool direct(const osm_loss_args* a) {
  return a->dtype == OSM_BF16 && a->D % 64 == 0 && (uintptr_t)a->weight % 16 == 0 && a->weight_stride % 8 == 0 &&
         a->weight_stride < kMaxRow;
}

// Whether a forward takes all tokens where they are: few, of rows that can be read there.
// (64 tokens of 256 over 1000 classes: two launches for three, 9.7 us for 13.4; 512 of 1024 over 32768:
// 42 us for 45; 1024: 80 both ways, 73 and 74 where 30% of the tokens do not count, and compacting gains from there on.)
bool in_place(const osm_loss_args* a) {
  return a->N <= 512 && a->dtype == OSM_BF16 && a->D % 64 == 0 && (uintptr_t)a->hidden % 16 == 0 && a->hidden_stride % 8 == 0 &&
         a->hidden_stride < kMaxRow;
}

// What a launch works on: the compacted hidden rows, and pieces of the vocabulary.
struct Plan {
  int64_t Npad, Dpad, parts, p_parts, piece;   // piece: classes, a multiple of kLossPad
  int splits, rows;                            // rows: classes of a forward's tile of logits
  bool direct;
};

// Classes of a piece: its parts of P, and of the weights where they are copied, are each at most
// 9 2^24 elements, unless 256 classes are more (less than 2^27: too few for 256 tiles of dW at
// 8192 tokens of 1024, 8% slower; twice and four times as many: the same; the ninth is for a last
// piece that is a little longer).  `rows`: elements of a class.
int64_t piece_of(int64_t V, int64_t rows) {
  const int64_t most = std::min((int64_t(9) << 24) / rows, kMaxRow - 1) / kLossPad * kLossPad;
  return std::min(std::max<int64_t>(most, kLossPad), up(V, kLossPad));
}

// Classes of 256 tiles of dW, a tile for every CU.
int64_t wave_of(int64_t D) { return std::max<int64_t>(1, 256 / ((D + 255) / 256)) * 256; }

// The classes of the next of `left`: all, or as many times 256 tiles of dW as a piece holds.
int64_t next_piece(int64_t left, int64_t piece, int64_t D) {
  const int64_t wave = wave_of(D);
  return left <= piece ? left : piece > wave ? piece / wave * wave : piece;
}

Plan plan_of(const osm_loss_args* a, bool bwd) {
  Plan n;
  n.parts = a->dtype == OSM_F32 ? 3 : 1;
  // (P rounded to bf16 puts a gradient off by 0.0002 to 0.0013 of its size, whatever the number
  // of tokens, where its own rounding puts it off by 0.0017: together 0.0018 for 65 tokens of 256
  // over 5000 classes, 0.0021 for 300 of 64 over 50.  A second part doubles both products; of few
  // tokens, whose products are bounded by the weights' bytes, it is held to twice the bits.)
  n.p_parts = n.parts == 1 && a->N <= 64 ? 2 : n.parts;
  n.Npad = up(std::max<int64_t>(a->N, 1), kLossPad);
  n.Dpad = up(a->D, 64);
  n.direct = direct(a);
  const int64_t across = (a->D + 255) / 256;
  // (a forward's launch has at most 2^32 threads, 256 for 64 x 64)
  const int64_t most = std::max<int64_t>((int64_t(1) << 36) / n.Npad / kLossPad * kLossPad - kLossPad, kLossPad);
  const int64_t copied = n.direct ? up(a->V, kLossPad) : piece_of(a->V, n.Dpad * n.parts);
  n.piece = std::min(copied, bwd ? piece_of(a->V, n.Npad * n.p_parts) : most);
  // Splits of dH's classes: as many as leave each a product that is worth its sums, six times the
  // work a class in three parts.  (1024 and 512 classes: fp32, 1000 x 7000 x 400, a backward in 187
  // and 179 us, 300 x 2000 x 800 in 71 and 64; bf16, 1500 x 4000 x 1024, in 81 and 86.)
  const int64_t tiles = across * (n.Npad / 256), least = n.parts == 1 ? 1024 : 512;
  n.splits = (int)std::max<int64_t>(1, std::min<int64_t>({256 / std::max<int64_t>(1, tiles), n.piece / least, 8}));
  LossParams p{};
  p.N = a->N;
  p.V = a->V;
  p.parts = (int)n.parts;
  p.p_parts = (int)n.p_parts;
  n.rows = osm::loss_tile_rows(p);
  return n;
}

// A forward's tiles along the vocabulary.
int tiles_of(const osm_loss_args* a, const Plan& n) { return (int)((a->V + n.rows - 1) / n.rows); }

// The regions of a workspace, each at a multiple of 256 bytes.
struct Regions {
  size_t total = 0;
  size_t add(size_t bytes) {
    const size_t at = total;
    total += (bytes + 255) / 256 * 256;
    return at;
  }
};
struct Layout {
  size_t targets, factors, places, count, h, w, own, stat, p, dh, total;
};
Layout layout_of(const osm_loss_args* a, const Plan& n, bool bwd) {
  Regions r;
  Layout l{};
  l.targets = r.add(a->N * 4);
  l.factors = r.add(bwd ? a->N * 8 : 0);
  l.places = r.add(a->N * 4);
  l.count = r.add(4);
  const size_t hidden = (size_t)n.parts * n.Npad * n.Dpad * 2;
  l.h = r.add(hidden);
  l.w = r.add(n.direct ? 0 : (size_t)n.parts * n.piece * n.Dpad * 2);
  if (!bwd) {
    l.own = r.add(n.Npad * 4);
    l.stat = r.add((size_t)tiles_of(a, n) * n.Npad * 8);
  } else {
    l.p = r.add((size_t)n.p_parts * n.Npad * n.piece * 2);
    l.dh = r.add((size_t)n.splits * n.Npad * n.Dpad * 4);
  }
  l.total = r.total;
  return l;
}

int check_workspace(const void* w, size_t have, size_t need) {
  if (!w || (uintptr_t)w % 256 || have < need)
    return fail(OSM_E_WORKSPACE, "the workspace must be 256-byte aligned and have %zu bytes (it has %zu)", need, w ? have : 0);
  return OSM_OK;
}

LossParams params_of(const osm_loss_args* a, const Plan& n, const Layout& l, void* workspace) {
  char* const w = static_cast<char*>(workspace);
  LossParams p{};
  p.N = a->N;
  p.D = a->D;
  p.V = a->V;
  p.Npad = (int)n.Npad;
  p.Dpad = (int)n.Dpad;
  p.parts = (int)n.parts;
  p.p_parts = (int)n.p_parts;
  p.hidden = a->hidden;
  p.hidden_s = a->hidden_stride;
  p.weight = a->weight;
  p.weight_s = a->weight_stride;
  p.targets = a->targets;
  p.ignore = a->ignore_index;
  p.tok = {reinterpret_cast<int*>(w + l.targets), reinterpret_cast<float2*>(w + l.factors), reinterpret_cast<int*>(w + l.places),
           reinterpret_cast<int*>(w + l.count)};
  p.h = reinterpret_cast<__bf16*>(w + l.h);
  p.h_ld = n.Dpad;
  p.h_part = n.Npad * n.Dpad;
  p.h_rows = (int)n.Npad;
  p.lse = a->lse;
  return p;
}

// The piece of vn classes from v0 on.
void set_piece(LossParams& p, const osm_loss_args* a, const Plan& n, const Layout& l, char* w, int64_t v0, int64_t vn) {
  p.v0 = v0;
  p.vn = (int)vn;
  p.vpad = (int)up(p.vn, kLossPad);
  p.w = n.direct ? static_cast<const __bf16*>(a->weight) + v0 * a->weight_stride : reinterpret_cast<const __bf16*>(w + l.w);
  p.w_ld = n.direct ? a->weight_stride : n.Dpad;
  p.w_part = n.direct ? 0 : (int64_t)p.vn * n.Dpad;
}

int hip_rc(hipError_t e) { return e == hipSuccess ? ok() : fail(OSM_E_HIP, "cross entropy launch: %s", hipGetErrorString(e)); }

hipError_t forward(const osm_loss_args* a, const Plan& n, const Layout& l, void* workspace, hipStream_t st) {
  char* const w = static_cast<char*>(workspace);
  LossParams p = params_of(a, n, l, workspace);
  p.own = reinterpret_cast<float*>(w + l.own);
  p.stat = reinterpret_cast<float2*>(w + l.stat);
  p.losses = a->losses;
  p.loss = a->loss;
  p.count = a->count;
  p.mean = (a->flags & OSM_LOSS_MEAN) != 0;
  __bf16* const parts = n.direct ? nullptr : reinterpret_cast<__bf16*>(w + l.w);
  hipError_t e = hipSuccess;
  bool packed = n.direct;
  set_piece(p, a, n, l, w, 0, std::min(n.piece, a->V));
  if (in_place(a)) {
    p.tok = {};
    p.h = static_cast<const __bf16*>(a->hidden);
    p.h_ld = a->hidden_stride;
    p.h_rows = (int)a->N;
  } else {
    e = osm::launch_loss_rows(p, reinterpret_cast<__bf16*>(w + l.h), parts, a->dtype, false, st);
    packed = true;
  }
  if (e != hipSuccess) return e;
  for (int64_t v0 = 0; v0 < a->V; v0 += n.piece, packed = n.direct) {
    p.tile0 = (int)(v0 / n.rows);
    set_piece(p, a, n, l, w, v0, std::min(n.piece, a->V - v0));
    if ((!packed && (e = osm::launch_loss_weight(p, parts, a->dtype, st)) != hipSuccess) || (e = osm::launch_loss_logits(p, st)) != hipSuccess)
      return e;
  }
  return osm::launch_loss_join(p, tiles_of(a, n), st);
}

hipError_t backward(const osm_loss_args* a, const osm_loss_bwd_args* b, const Plan& n, const Layout& l, void* workspace, hipStream_t st) {
  char* const w = static_cast<char*>(workspace);
  LossParams p = params_of(a, n, l, workspace);
  p.p = reinterpret_cast<__bf16*>(w + l.p);
  p.dh = reinterpret_cast<float*>(w + l.dh);
  p.splits = n.splits;
  p.grad = b->grad;
  p.grad_losses = b->grad_losses;
  p.count_in = b->count;
  p.grad_h = b->grad_hidden;
  p.grad_w = b->grad_weight;
  __bf16* const parts = n.direct ? nullptr : reinterpret_cast<__bf16*>(w + l.w);
  hipError_t e;
  for (int64_t v0 = 0, vn; v0 < a->V; v0 += vn) {
    vn = next_piece(a->V - v0, n.piece, a->D);
    p.first = v0 == 0;
    set_piece(p, a, n, l, w, v0, vn);
    if (p.first)
      e = osm::launch_loss_rows(p, reinterpret_cast<__bf16*>(w + l.h), parts, a->dtype, true, st);
    else
      e = n.direct ? hipSuccess : osm::launch_loss_weight(p, parts, a->dtype, st);
    if (e != hipSuccess || (e = osm::launch_loss_probs(p, st)) != hipSuccess) return e;
    if (b->grad_hidden && (e = osm::launch_loss_dh(p, st)) != hipSuccess) return e;
    if (!b->grad_weight) continue;
    // (what is over 256 tiles of dW, in tiles of its own: 17233 classes, 8192 tokens, 1024 columns: 338 us in one launch
    // of 280 tiles, 254 and 52 in two)
    const int64_t wave = wave_of(a->D), whole = n.parts == 1 && vn > wave ? vn / wave * wave : vn;
    if ((e = osm::launch_loss_dw(p, 0, (int)whole, st)) != hipSuccess) return e;
    if (whole < vn && (e = osm::launch_loss_dw(p, (int)whole, (int)(vn - whole), st)) != hipSuccess) return e;
  }
  return b->grad_hidden ? osm::launch_loss_finish(p, a->dtype, st) : hipSuccess;
}

}  // namespace

extern "C" {

size_t osm_linear_ce_workspace_bytes(const osm_loss_args* a) {
  return check_args(a) == OSM_OK && a->N > 0 ? layout_of(a, plan_of(a, false), false).total : 0;
}

int osm_linear_ce_fwd(const osm_loss_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_args(a);
  if (rc != OSM_OK) return rc;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const void* words[3] = {a->losses, a->loss, a->count};
  for (const void* w : words)
    if ((uintptr_t)w % 4) return fail(OSM_E_LAYOUT, "losses, loss and count must be 4-byte aligned");
  if ((a->loss && !a->losses && a->N > 0) || (a->count && !a->loss)) return fail(OSM_E_ARG, "loss without losses, or count without loss");
  if (a->N == 0) return a->loss ? hip_rc(osm::launch_loss_none(a->loss, a->count, st)) : ok();
  if ((rc = check_inputs(a)) != OSM_OK) return rc;
  const Plan n = plan_of(a, false);
  const Layout l = layout_of(a, n, false);
  if ((rc = check_workspace(workspace, workspace_bytes, l.total)) != OSM_OK) return rc;
  return hip_rc(forward(a, n, l, workspace, st));
}

size_t osm_linear_ce_bwd_workspace_bytes(const osm_loss_args* a) {
  return check_args(a) == OSM_OK && a->N > 0 ? layout_of(a, plan_of(a, true), true).total : 0;
}

int osm_linear_ce_bwd(const osm_loss_args* a, const osm_loss_bwd_args* b, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_args(a);
  if (rc != OSM_OK) return rc;
  if (!b) return fail(OSM_E_ARG, "bwd is NULL");
  const void* words[3] = {b->grad, b->grad_losses, b->count};
  for (const void* w : words)
    if ((uintptr_t)w % 4) return fail(OSM_E_LAYOUT, "grad, grad_losses and count must be 4-byte aligned");
  // (rows of whole 4-element units are written by them)
  const int es = a->dtype == OSM_F32 ? 4 : 2, unit = a->D % 4 == 0 ? 4 * es : es;
  if ((uintptr_t)b->grad_hidden % unit || (uintptr_t)b->grad_weight % unit)
    return fail(OSM_E_LAYOUT, "grad_hidden and grad_weight must be aligned to %d bytes", unit);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (a->N == 0)
    return b->grad_weight ? hip_rc(osm::launch_loss_zero(b->grad_weight, a->V * a->D, a->dtype, st)) : ok();
  if ((rc = check_inputs(a)) != OSM_OK) return rc;
  const Plan n = plan_of(a, true);
  const Layout l = layout_of(a, n, true);
  if ((rc = check_workspace(workspace, workspace_bytes, l.total)) != OSM_OK) return rc;
  return hip_rc(backward(a, b, n, l, workspace, st));
}

}  // extern "C"
