// C ABI of the layer norm and of gradient clipping: argument checks and
// dispatch.  Declared in include/osm.h.
#include <algorithm>
#include <new>
#include <utility>
#include <vector>

#include "osm.h"
#include "osm_kernels.h"
#include "osm_norm.h"

namespace {

using osm::ClipTable;
using osm::fail;
using osm::NormParams;
using osm::ok;

int check_norm(const osm_norm_args* a) {
  if (!a) return fail(OSM_E_ARG, "args is NULL");
  if (a->abi_version != OSM_ABI_VERSION)
    return fail(OSM_E_ARG, "abi_version %d does not match library ABI %d", a->abi_version, OSM_ABI_VERSION);
  if (a->dtype != OSM_F32 && a->dtype != OSM_BF16) return fail(OSM_E_DTYPE, "dtype %d unsupported", a->dtype);
  if (a->rows < 0 || a->D < 1 || a->D >= (int64_t(1) << 31))
    return fail(OSM_E_SHAPE, "rows=%lld must be >= 0 and D=%lld in [1, 2^31)", (long long)a->rows, (long long)a->D);
  if (!(a->eps >= 0.0f)) return fail(OSM_E_ARG, "eps=%g must be >= 0", (double)a->eps);
  const void* words[4] = {a->weight, a->bias, a->mean, a->rstd};
  for (const void* w : words)
    if ((uintptr_t)w % 4) return fail(OSM_E_LAYOUT, "weight, bias, mean and rstd must be 4-byte aligned");
  if (!a->mean != !a->rstd) return fail(OSM_E_ARG, "mean and rstd go together");
  return OSM_OK;
}

int check_matrix(const void* p, int64_t stride, int64_t least, int esize, const char* name) {
  if (!p) return fail(OSM_E_ARG, "%s is NULL", name);
  if ((uintptr_t)p % esize) return fail(OSM_E_LAYOUT, "%s is not aligned to its elements", name);
  if (stride < least) return fail(OSM_E_LAYOUT, "%s: row stride %lld below %lld", name, (long long)stride, (long long)least);
  return OSM_OK;
}

bool whole(const void* p, int64_t stride, int esize) { return (uintptr_t)p % 16 == 0 && stride * esize % 16 == 0; }

NormParams params_of(const osm_norm_args* a) {
  NormParams p{};
  p.x = a->x;
  p.x_stride = a->x_stride;
  p.weight = a->weight;
  p.bias = a->bias;
  p.mean = a->mean;
  p.rstd = a->rstd;
  p.rows = a->rows;
  p.D = a->D;
  p.eps = a->eps;
  return p;
}

int check_clip(const osm_clip_args* a) {
  if (!a) return fail(OSM_E_ARG, "args is NULL");
  if (a->abi_version != OSM_ABI_VERSION)
    return fail(OSM_E_ARG, "abi_version %d does not match library ABI %d", a->abi_version, OSM_ABI_VERSION);
  if (a->flags & ~OSM_CLIP_SCALE) return fail(OSM_E_ARG, "unknown flag bits 0x%x", a->flags);
  if (a->count < 0 || a->count > (1 << 24)) return fail(OSM_E_SHAPE, "count=%lld outside [0, 2^24]", (long long)a->count);
  if (a->count > 0 && (!a->tensors || !a->sizes || !a->dtypes))
    return fail(OSM_E_ARG, "tensors, sizes and dtypes must be non-NULL");
  for (int64_t i = 0; i < a->count; ++i) {
    if (a->dtypes[i] != OSM_F32 && a->dtypes[i] != OSM_BF16)
      return fail(OSM_E_DTYPE, "tensor %lld: dtype %d unsupported", (long long)i, a->dtypes[i]);
    // (a launch's chunks are counted in 31 bits)
    if (a->sizes[i] < 0 || a->sizes[i] > (int64_t(1) << 40))
      return fail(OSM_E_SHAPE, "tensor %lld: %lld elements outside [0, 2^40]", (long long)i, (long long)a->sizes[i]);
    if (a->sizes[i] > 0 && !a->tensors[i]) return fail(OSM_E_ARG, "tensor %lld is NULL", (long long)i);
    if ((uintptr_t)a->tensors[i] % (a->dtypes[i] == OSM_F32 ? 4 : 2))
      return fail(OSM_E_LAYOUT, "tensor %lld is not aligned to its elements", (long long)i);
  }
  if (!(a->max_norm >= 0.0) || !(a->eps >= 0.0))
    return fail(OSM_E_ARG, "max_norm=%g and eps=%g must be >= 0", a->max_norm, a->eps);
  return OSM_OK;
}

// Tensors that are scaled in place share no memory: two workgroups would read and
// write the same elements in no order.
int check_apart(const osm_clip_args* a) try {
  std::vector<std::pair<uintptr_t, uintptr_t>> spans;
  spans.reserve(a->count);
  for (int64_t i = 0; i < a->count; ++i) {
    const uintptr_t p = (uintptr_t)a->tensors[i];
    if (a->sizes[i] > 0) spans.emplace_back(p, p + (uintptr_t)a->sizes[i] * (a->dtypes[i] == OSM_F32 ? 4 : 2));
  }
  std::sort(spans.begin(), spans.end());
  for (size_t i = 1; i < spans.size(); ++i)
    if (spans[i].first < spans[i - 1].second)
      return fail(OSM_E_LAYOUT, "two of the tensors share memory, at %p", (void*)spans[i].first);
  return OSM_OK;
} catch (const std::bad_alloc&) {
  return fail(OSM_E_ARG, "no host memory for %lld tensors", (long long)a->count);
}

int64_t chunks_of(int64_t n) { return (n + osm::kClipChunk - 1) / osm::kClipChunk; }

// Calls f(table) for the launches that cover the tensors (at least one, so that
// the norm of none is written): up to 150 tensors and 2^30 chunks each.
template <typename F>
int for_tables(const osm_clip_args* a, F f) {
  int64_t i = 0, part0 = 0;
  do {
    ClipTable t;
    int64_t chunks = 0;
    t.count = 0;
    t.first[0] = 0;
    for (; i < a->count && t.count < osm::kClipTensors; ++i) {
      if (a->sizes[i] == 0) continue;
      const int64_t n = chunks_of(a->sizes[i]);
      if (chunks + n > (1 << 30)) break;
      const int k = t.count++;
      t.p[k] = a->tensors[i];
      t.n[k] = a->sizes[i];
      t.bf16[k] = a->dtypes[i] == OSM_BF16;
      t.vec[k] = (uintptr_t)a->tensors[i] % 16 == 0;
      chunks += n;
      t.first[k + 1] = (int)chunks;
    }
    t.part0 = (int)part0;
    t.parts = (int)std::min<int64_t>(chunks, osm::kClipMaxGroups);
    part0 += t.parts;
    const int rc = f(t);
    if (rc != OSM_OK) return rc;
  } while (i < a->count);
  return OSM_OK;
}

}  // namespace

extern "C" {

int osm_layer_norm_fwd(const osm_norm_args* a, void* stream) {
  int rc = check_norm(a);
  if (rc != OSM_OK || a->rows == 0) return rc == OSM_OK ? ok() : rc;
  const int es = a->dtype == OSM_F32 ? 4 : 2;
  if ((rc = check_matrix(a->x, a->x_stride, 0, es, "x")) != OSM_OK ||
      (rc = check_matrix(a->y, a->y_stride, a->rows > 1 ? a->D : 0, es, "y")) != OSM_OK)
    return rc;
  NormParams p = params_of(a);
  p.y = a->y;
  p.y_stride = a->y_stride;
  p.vec = a->D * es % 16 == 0 && whole(a->x, a->x_stride, es) && whole(a->y, a->y_stride, es);
  const hipError_t e = osm::launch_layer_norm_fwd(p, a->dtype, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? ok() : fail(OSM_E_HIP, "layer norm launch: %s", hipGetErrorString(e));
}

size_t osm_layer_norm_bwd_workspace_bytes(const osm_norm_args* a) {
  if (check_norm(a) != OSM_OK || a->rows == 0) return 0;
  return (size_t)osm::norm_lines(a->rows, a->D) * 2 * a->D * sizeof(float);
}

int osm_layer_norm_bwd(const osm_norm_args* a, const osm_norm_bwd_args* b, void* workspace, size_t workspace_bytes,
                       void* stream) {
  int rc = check_norm(a);
  if (rc != OSM_OK) return rc;
  if (!b) return fail(OSM_E_ARG, "bwd is NULL");
  if ((uintptr_t)b->grad_weight % 4 || (uintptr_t)b->grad_bias % 4)
    return fail(OSM_E_LAYOUT, "grad_weight and grad_bias must be 4-byte aligned");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (a->rows == 0) {
    hipError_t e = hipSuccess;
    if (b->grad_weight) e = osm::launch_fill_zero(b->grad_weight, a->D * sizeof(float), st);
    if (e == hipSuccess && b->grad_bias) e = osm::launch_fill_zero(b->grad_bias, a->D * sizeof(float), st);
    return e == hipSuccess ? ok() : fail(OSM_E_HIP, "gradient fill launch: %s", hipGetErrorString(e));
  }
  const int es = a->dtype == OSM_F32 ? 4 : 2;
  if (!a->mean) return fail(OSM_E_ARG, "mean and rstd are NULL");
  if ((rc = check_matrix(a->x, a->x_stride, 0, es, "x")) != OSM_OK ||
      (rc = check_matrix(b->grad_y, b->grad_y_stride, 0, es, "grad_y")) != OSM_OK ||
      (b->grad_x && (rc = check_matrix(b->grad_x, b->grad_x_stride, a->rows > 1 ? a->D : 0, es, "grad_x")) != OSM_OK))
    return rc;
  const size_t need = osm_layer_norm_bwd_workspace_bytes(a);
  if (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < need)
    return fail(OSM_E_WORKSPACE, "the workspace must be 256-byte aligned and have %zu bytes (it has %zu)", need,
                workspace ? workspace_bytes : 0);
  NormParams p = params_of(a);
  p.gy = b->grad_y;
  p.gy_stride = b->grad_y_stride;
  p.gx = b->grad_x;
  p.gx_stride = b->grad_x_stride;
  p.part = static_cast<float*>(workspace);
  p.vec = a->D * es % 16 == 0 && whole(a->x, a->x_stride, es) && whole(b->grad_y, b->grad_y_stride, es) &&
          (!b->grad_x || whole(b->grad_x, b->grad_x_stride, es));
  const hipError_t e = osm::launch_layer_norm_bwd(p, b->grad_weight, b->grad_bias, a->dtype, st);
  return e == hipSuccess ? ok() : fail(OSM_E_HIP, "layer norm backward launch: %s", hipGetErrorString(e));
}

size_t osm_clip_workspace_bytes(const osm_clip_args* a) {
  if (check_clip(a) != OSM_OK) return 0;
  size_t parts = 0;
  for_tables(a, [&](const ClipTable& t) {
    parts += t.parts;
    return OSM_OK;
  });
  return std::max<size_t>(parts, 1) * sizeof(double);
}

int osm_clip_grad_norm(const osm_clip_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_clip(a);
  if (rc == OSM_OK && a->flags & OSM_CLIP_SCALE) rc = check_apart(a);
  if (rc != OSM_OK) return rc;
  if (!a->norm || (uintptr_t)a->norm % 4) return fail(OSM_E_ARG, "norm is NULL or not 4-byte aligned");
  const size_t need = osm_clip_workspace_bytes(a);
  if (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < need)
    return fail(OSM_E_WORKSPACE, "the workspace must be 256-byte aligned and have %zu bytes (it has %zu)", need,
                workspace ? workspace_bytes : 0);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  double* const part = static_cast<double*>(workspace);
  int parts = 0;
  rc = for_tables(a, [&](const ClipTable& t) {
    parts += t.parts;
    const hipError_t e = t.parts ? osm::launch_clip_sums(t, part, st) : hipSuccess;
    return e == hipSuccess ? (int)OSM_OK : fail(OSM_E_HIP, "norm launch: %s", hipGetErrorString(e));
  });
  if (rc != OSM_OK) return rc;
  const bool scale = a->flags & OSM_CLIP_SCALE;
  float* norm = a->norm;   // written by the first launch
  return for_tables(a, [&](const ClipTable& t) {
    if (!norm && (!scale || !t.parts)) return ok();
    const hipError_t e = osm::launch_clip_scale(t, part, parts, a->max_norm, a->eps, norm, scale && t.parts, st);
    norm = nullptr;
    return e == hipSuccess ? ok() : fail(OSM_E_HIP, "clip launch: %s", hipGetErrorString(e));
  });
}

}  // extern "C"
