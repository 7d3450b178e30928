// C ABI of the residual norm: argument checks and dispatch.  Declared in
// include/osm.h.
#include "osm.h"
#include "osm_kernels.h"
#include "osm_norm.h"
#include "osm_resnorm.h"

namespace {

using osm::fail;
using osm::ok;
using osm::ResnormParams;

int size_of(int dtype) { return dtype == OSM_F32 ? 4 : 2; }

int check_args(const osm_resnorm_args* a) {
  if (!a) return fail(OSM_E_ARG, "args is NULL");
  if (a->abi_version != OSM_ABI_VERSION)
    return fail(OSM_E_ARG, "abi_version %d does not match library ABI %d", a->abi_version, OSM_ABI_VERSION);
  if (a->flags & ~(OSM_RESNORM_NORM_Y | OSM_RESNORM_RMS)) return fail(OSM_E_ARG, "unknown flag bits 0x%x", a->flags);
  const int s = a->stream_dtype, b = a->block_dtype;
  if ((s != OSM_F32 && s != OSM_BF16) || (b != OSM_F32 && b != OSM_BF16) || (b == OSM_F32 && s != OSM_F32))
    return fail(OSM_E_DTYPE, "stream_dtype %d with block_dtype %d unsupported", s, b);
  if (a->rows < 0 || a->D < 1 || a->D > (int64_t(1) << 25))   // (threads of the sums' launch: 96 D)
    return fail(OSM_E_SHAPE, "rows=%lld must be >= 0 and D=%lld in [1, 2^25]", (long long)a->rows, (long long)a->D);
  if (!(a->eps >= 0.0f)) return fail(OSM_E_ARG, "eps=%g must be >= 0", (double)a->eps);
  const void* words[4] = {a->scale, a->weight, a->bias, a->stats};
  for (const void* w : words)
    if ((uintptr_t)w % 4) return fail(OSM_E_LAYOUT, "scale, weight, bias and stats must be 4-byte aligned");
  return OSM_OK;
}

// `least`: the row stride has to be at least that.
int check_matrix(const void* p, int64_t stride, int64_t least, int esize, const char* name) {
  if (!p) return fail(OSM_E_ARG, "%s is NULL", name);
  if ((uintptr_t)p % esize) return fail(OSM_E_LAYOUT, "%s is not aligned to its elements", name);
  if (stride < least) return fail(OSM_E_LAYOUT, "%s: row stride %lld below %lld", name, (long long)stride, (long long)least);
  return OSM_OK;
}

// (absent matrices are in every form)
bool whole(const void* p, int64_t stride, int esize) { return !p || ((uintptr_t)p % 16 == 0 && stride * esize % 16 == 0); }

int check_inputs(const osm_resnorm_args* a) {
  const int xs = size_of(a->stream_dtype), ys = size_of(a->block_dtype);
  int rc = check_matrix(a->x, a->x_stride, 0, xs, "x");
  if (rc == OSM_OK) rc = check_matrix(a->y, a->y_stride, 0, ys, "y");
  if (rc == OSM_OK && a->gate) rc = check_matrix(a->gate, a->gate_stride, 0, ys, "gate");
  return rc;
}

ResnormParams params_of(const osm_resnorm_args* a) {
  ResnormParams p{};
  p.x = a->x;
  p.y = a->y;
  p.gate = a->gate;
  p.x_s = a->x_stride;
  p.y_s = a->y_stride;
  p.gate_s = a->gate_stride;
  p.scale = a->scale;
  p.weight = a->weight;
  p.bias = a->bias;
  p.stats = a->stats;
  p.rows = a->rows;
  p.D = a->D;
  p.eps = a->eps;
  p.norm_y = (a->flags & OSM_RESNORM_NORM_Y) != 0;
  p.rms = (a->flags & OSM_RESNORM_RMS) != 0;
  const int xs = size_of(a->stream_dtype), ys = size_of(a->block_dtype);
  p.vec = a->D * ys % 16 == 0 && whole(a->x, a->x_stride, xs) && whole(a->y, a->y_stride, ys) && whole(a->gate, a->gate_stride, ys);
  return p;
}

}  // namespace

extern "C" {

int osm_residual_norm_fwd(const osm_resnorm_args* a, void* stream) {
  int rc = check_args(a);
  if (rc != OSM_OK || a->rows == 0) return rc == OSM_OK ? ok() : rc;
  const int xs = size_of(a->stream_dtype), ys = size_of(a->block_dtype);
  const int64_t least = a->rows > 1 ? a->D : 0;
  if ((rc = check_inputs(a)) != OSM_OK || (rc = check_matrix(a->r, a->r_stride, least, xs, "r")) != OSM_OK ||
      (rc = check_matrix(a->n, a->n_stride, least, ys, "n")) != OSM_OK)
    return rc;
  ResnormParams p = params_of(a);
  p.r = a->r;
  p.n = a->n;
  p.r_s = a->r_stride;
  p.n_s = a->n_stride;
  p.vec = p.vec && whole(a->r, a->r_stride, xs) && whole(a->n, a->n_stride, ys);
  const hipError_t e = osm::launch_resnorm_fwd(p, a->stream_dtype, a->block_dtype, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? ok() : fail(OSM_E_HIP, "residual norm launch: %s", hipGetErrorString(e));
}

size_t osm_residual_norm_bwd_workspace_bytes(const osm_resnorm_args* a) {
  if (check_args(a) != OSM_OK || a->rows == 0) return 0;
  const size_t lines = (size_t)osm::norm_lines(a->rows, a->D) * 3 * a->D;
  return (lines + (osm::resnorm_long(a->D) ? 2 * (size_t)a->rows : 0)) * sizeof(float);
}

int osm_residual_norm_bwd(const osm_resnorm_args* a, const osm_resnorm_bwd_args* b, void* workspace, size_t workspace_bytes,
                          void* stream) {
  int rc = check_args(a);
  if (rc != OSM_OK) return rc;
  if (!b) return fail(OSM_E_ARG, "bwd is NULL");
  float* const sums[3] = {b->grad_weight, b->grad_bias, b->grad_scale};
  for (float* s : sums)
    if ((uintptr_t)s % 4) return fail(OSM_E_LAYOUT, "grad_weight, grad_bias and grad_scale must be 4-byte aligned");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (a->rows == 0) {
    for (float* s : sums) {
      const hipError_t e = s ? osm::launch_fill_zero(s, a->D * sizeof(float), st) : hipSuccess;
      if (e != hipSuccess) return fail(OSM_E_HIP, "gradient fill launch: %s", hipGetErrorString(e));
    }
    return ok();
  }
  const int xs = size_of(a->stream_dtype), ys = size_of(a->block_dtype);
  const int64_t least = a->rows > 1 ? a->D : 0;
  if (!a->stats) return fail(OSM_E_ARG, "stats is NULL");
  if (b->grad_gate && !a->gate) return fail(OSM_E_ARG, "grad_gate without a gate");
  if ((rc = check_inputs(a)) != OSM_OK ||
      (b->grad_r && (rc = check_matrix(b->grad_r, b->grad_r_stride, 0, xs, "grad_r")) != OSM_OK) ||
      (b->grad_n && (rc = check_matrix(b->grad_n, b->grad_n_stride, 0, ys, "grad_n")) != OSM_OK) ||
      (b->grad_x && (rc = check_matrix(b->grad_x, b->grad_x_stride, least, xs, "grad_x")) != OSM_OK) ||
      (b->grad_y && (rc = check_matrix(b->grad_y, b->grad_y_stride, least, ys, "grad_y")) != OSM_OK) ||
      (b->grad_gate && (rc = check_matrix(b->grad_gate, b->grad_gate_stride, least, ys, "grad_gate")) != OSM_OK))
    return rc;
  const size_t need = osm_residual_norm_bwd_workspace_bytes(a);
  if (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < need)
    return fail(OSM_E_WORKSPACE, "the workspace must be 256-byte aligned and have %zu bytes (it has %zu)", need,
                workspace ? workspace_bytes : 0);
  ResnormParams p = params_of(a);
  p.gr = b->grad_r;
  p.gn = b->grad_n;
  p.gx = b->grad_x;
  p.gy = b->grad_y;
  p.gg = b->grad_gate;
  p.gr_s = b->grad_r_stride;
  p.gn_s = b->grad_n_stride;
  p.gx_s = b->grad_x_stride;
  p.gy_s = b->grad_y_stride;
  p.gg_s = b->grad_gate_stride;
  p.part = static_cast<float*>(workspace);
  p.sums = p.part + (size_t)osm::norm_lines(a->rows, a->D) * 3 * a->D;
  p.vec = p.vec && whole(p.gr, p.gr_s, xs) && whole(p.gn, p.gn_s, ys) && whole(p.gx, p.gx_s, xs) && whole(p.gy, p.gy_s, ys) &&
          whole(p.gg, p.gg_s, ys);
  const hipError_t e = osm::launch_resnorm_bwd(p, b->grad_weight, b->grad_bias, b->grad_scale, a->stream_dtype, a->block_dtype, st);
  return e == hipSuccess ? ok() : fail(OSM_E_HIP, "residual norm backward launch: %s", hipGetErrorString(e));
}

}  // extern "C"
