// Launch path of the torch-facing operators (orthossm_amd/ops.py) in native
// code: reads the tensors, fills the C ABI's argument structs, allocates the
// outputs and launches.  Each function serves the form its kernel takes as it
// stands (tensors of the right dtype, device and layout) and returns None for
// anything else, which the Python function of the same name then converts or
// refuses; arguments, defaults and results are the Python function's.
//
// What it replaces: the same steps through ctypes, 12 us of host time a
// forward call against 5 (measured on an MI355X host, B=1 S=16), longer than
// the kernels themselves run at short sequences.
//
// Nothing is kept between calls: workspaces come from the Python module's own
// cache, the stream is read on every call.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include <cmath>
#include <vector>

#include "osm.h"

namespace {

// Set by init(): the library's functions (the instance ctypes has loaded) and
// the Python module's helpers.
struct Lib {
  decltype(&osm_workspace_bytes) workspace_bytes;
  decltype(&osm_cheby_ema_fwd) fwd;
  decltype(&osm_cheby_ema_ttt) ttt;
  decltype(&osm_cheby_ema_bwd) bwd;
  decltype(&osm_v10_chunked_ttt) v10;
  decltype(&osm_v10_bwd) v10_bwd;
  decltype(&osm_lut_fwd_workspace_bytes) lut_bytes;
  decltype(&osm_cheby_ema_lut_fwd_ws) lut_ws;
  decltype(&osm_engine_scratch_bytes) engine_bytes;
  decltype(&osm_engine_prologue) engine;
  int (*stream_is_capturing)(void* stream, int* status);   // hipStreamIsCapturing
  decltype(&osm_delta_saved_bytes) delta_saved;
  decltype(&osm_delta_workspace_bytes) delta_bytes;
  decltype(&osm_delta_fwd) delta_fwd;
  decltype(&osm_delta_bwd_workspace_bytes) delta_bwd_bytes;
  decltype(&osm_delta_bwd) delta_bwd;
  decltype(&osm_delta_step) delta_step;
  decltype(&osm_layer_norm_fwd) norm_fwd;
  decltype(&osm_layer_norm_bwd_workspace_bytes) norm_bwd_bytes;
  decltype(&osm_layer_norm_bwd) norm_bwd;
  decltype(&osm_clip_workspace_bytes) clip_bytes;
  decltype(&osm_clip_grad_norm) clip;
  decltype(&osm_gated_ema_saved_bytes) ema_saved;
  decltype(&osm_gated_ema_workspace_bytes) ema_bytes;
  decltype(&osm_gated_ema_fwd) ema_fwd;
  decltype(&osm_gated_ema_bwd_workspace_bytes) ema_bwd_bytes;
  decltype(&osm_gated_ema_bwd) ema_bwd;
  decltype(&osm_gated_ema_step) ema_step;
  decltype(&osm_residual_norm_fwd) block_fwd;
  decltype(&osm_residual_norm_bwd_workspace_bytes) block_bwd_bytes;
  decltype(&osm_residual_norm_bwd) block_bwd;
  decltype(&osm_linear_ce_workspace_bytes) loss_bytes;
  decltype(&osm_linear_ce_fwd) loss_fwd;
  decltype(&osm_linear_ce_bwd_workspace_bytes) loss_bwd_bytes;
  decltype(&osm_linear_ce_bwd) loss_bwd;
} lib;
constexpr int kFunctions = 35;
PyObject* raw_stream = nullptr;   // device index -> raw stream handle
PyObject* ws_cache = nullptr;     // {(device index, stream, op): uint8 tensor}
PyObject* workspace = nullptr;    // (device, stream, bytes, op) -> uint8 tensor
PyObject* check = nullptr;        // raises for a status code

constexpr int kOpLut = 3;

// Releases the GIL for a scope: allocations and launches may block.
struct NoGil {
  PyThreadState* s = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(s); }
};

// An owned reference.
struct Ref {
  PyObject* o = nullptr;
  ~Ref() { Py_XDECREF(o); }
};

const at::Tensor* plain(PyObject* o) {
  return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr;
}

bool is_f32(const at::Tensor& t) { return t.scalar_type() == at::kFloat; }
bool is_bf16(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16; }
int code(const at::Tensor& t) { return is_f32(t) ? OSM_F32 : OSM_BF16; }

// [B,S,D] rows as the kernels address them: lane stride 1, no negative stride.
bool rows(const at::Tensor& t, const at::Tensor& x) {
  return t.dim() == 3 && t.device() == x.device() && t.sizes() == x.sizes() && t.stride(2) == 1 && t.stride(0) >= 0 &&
         t.stride(1) >= 0;
}

bool f32_flat(const at::Tensor& t, int64_t n, const at::Tensor& x) {
  return is_f32(t) && t.device() == x.device() && t.numel() == n && t.is_contiguous();
}

bool f32_vec(const at::Tensor* t, int64_t n, const at::Tensor& x) {
  return t && t->dim() == 1 && f32_flat(*t, n, x);
}

float* fptr(const at::Tensor& t) { return static_cast<float*>(t.data_ptr()); }

at::Tensor empty(at::IntArrayRef size, const at::Tensor& like, at::ScalarType dtype) {
  return at::empty(size, like.options().dtype(dtype).requires_grad(false));
}

PyObject* fail_rc(int rc) {
  PyObject* r = PyObject_CallFunction(check, "i", rc);
  Py_XDECREF(r);
  if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "osm: launch failed");
  return nullptr;
}

// Current raw stream of x's device; false with a Python error set.
bool stream_of(const at::Tensor& x, Ref* obj, void** stream) {
  const Ref idx{PyLong_FromLong(x.get_device())};
  if (!idx.o) return false;
  obj->o = PyObject_CallFunctionObjArgs(raw_stream, idx.o, nullptr);
  if (!obj->o) return false;
  *stream = PyLong_AsVoidPtr(obj->o);
  return !PyErr_Occurred();
}

// The workspace of (device, stream, op), from the module's cache or, where it
// is to be made or a graph is to hold it, by its _workspace; false with a Python
// error set.
bool get_workspace(PyObject* x_obj, const at::Tensor& x, PyObject* stream, void* raw, size_t need, int op,
                   at::Tensor* ws) {
  PyObject* key = Py_BuildValue("(iOi)", (int)x.get_device(), stream, op);
  if (!key) return false;
  PyObject* hit = PyDict_GetItemWithError(ws_cache, key);
  Py_DECREF(key);
  if (hit && THPVariable_Check(hit) && (size_t)THPVariable_Unpack(hit).numel() >= need) {
    *ws = THPVariable_Unpack(hit);
    int status = 0;
    if (lib.stream_is_capturing(raw, &status) == 0 && status == 0) return true;
  }
  if (PyErr_Occurred()) return false;
  PyObject* dev = PyObject_GetAttrString(x_obj, "device");
  if (!dev) return false;
  PyObject* made = PyObject_CallFunction(workspace, "OOni", dev, stream, (Py_ssize_t)need, op);
  Py_DECREF(dev);
  if (!made) return false;
  *ws = THPVariable_Unpack(made);
  Py_DECREF(made);
  return true;
}

bool as_float(PyObject* o, float* v) {
  const double d = PyFloat_AsDouble(o);
  if (d == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  *v = (float)d;
  return true;
}

// An integer; false for what int() would have to convert (a float, say), which
// the Python path then does or refuses.
bool as_int(PyObject* o, int64_t* v) {
  *v = PyLong_AsLongLong(o);
  if (*v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

struct Common {
  const at::Tensor *x, *coeffs, *damping, *lam, *g = nullptr;
  osm_cheby_args a{};
  int64_t B, S, H, K, hd;
};

// args: x, coeffs, damping, lam, g, lam_shift, lam_min, lam_max, flags.
bool common(PyObject* const* p, Common* c) {
  c->x = plain(p[0]);
  c->coeffs = plain(p[1]);
  c->damping = plain(p[2]);
  c->lam = plain(p[3]);
  if (!c->x || !c->coeffs || !c->damping || !c->lam) return false;
  const at::Tensor &x = *c->x, &cf = *c->coeffs;
  if (!x.is_cuda() || !(is_f32(x) || is_bf16(x)) || !rows(x, x)) return false;
  if (cf.dim() != 4 || !is_f32(cf) || cf.device() != x.device() || cf.stride(3) != 1) return false;
  c->B = x.size(0);
  c->S = x.size(1);
  c->H = cf.size(1);
  c->K = cf.size(2);
  c->hd = cf.size(3);
  if (cf.size(0) != c->B || c->H * c->hd != x.size(2)) return false;
  if (!f32_vec(c->damping, c->H, x) || !f32_vec(c->lam, c->H, x)) return false;
  osm_cheby_args& a = c->a;
  if (p[4] != Py_None) {
    c->g = plain(p[4]);
    if (!c->g || !is_f32(*c->g) || c->g->device() != x.device() || c->g->dim() != 3 || c->g->size(0) != c->B ||
        c->g->size(1) != c->S || c->g->size(2) != c->H)
      return false;
    a.g = fptr(*c->g);
    a.g_stride_b = c->g->stride(0);
    a.g_stride_s = c->g->stride(1);
    a.g_stride_h = c->g->stride(2);
  }
  if (!as_float(p[5], &a.lam_shift) || !as_float(p[6], &a.lam_min) || !as_float(p[7], &a.lam_max)) return false;
  a.abi_version = OSM_ABI_VERSION;
  a.flags = (int32_t)PyLong_AsLong(p[8]);
  a.B = c->B;
  a.S = c->S;
  a.H = c->H;
  a.hd = c->hd;
  a.K = c->K;
  a.x = x.data_ptr();
  a.x_dtype = code(x);
  a.x_stride_b = x.stride(0);
  a.x_stride_s = x.stride(1);
  a.coeffs = fptr(cf);
  a.c_stride_b = cf.stride(0);
  a.c_stride_h = cf.stride(1);
  a.c_stride_k = cf.stride(2);
  a.damping = fptr(*c->damping);
  a.lam = fptr(*c->lam);
  return true;
}

// The output rows: `o` a caller's buffer or None, `dt` the dtype code.
bool out_rows(PyObject* o, int dt, Common* c, at::Tensor* out) {
  const at::ScalarType want = dt == OSM_F32 ? at::kFloat : at::kBFloat16;
  if (o != Py_None) {
    const at::Tensor* t = plain(o);
    if (!t || t->scalar_type() != want || !rows(*t, *c->x)) return false;
    *out = *t;
  }
  c->a.out_dtype = dt;
  return true;
}

void set_out(Common* c, const at::Tensor& out) {
  c->a.out = out.data_ptr();
  c->a.out_stride_b = out.stride(0);
  c->a.out_stride_s = out.stride(1);
}

// forward(<common 9>, ema_init, out_dtype, out, want_state, state_out) and
// ttt(.., state_out, target): None, or (out, ema_final | None) / (out, grad, ema_final | None).
PyObject* run_forward(PyObject* const* p, bool ttt) {
  Common c;
  const int target = ttt ? (int)PyLong_AsLong(p[14]) : 0;
  if (!common(p, &c)) Py_RETURN_NONE;
  const at::Tensor& x = *c.x;
  const int64_t D = c.H * c.hd;
  if (p[9] != Py_None) {
    const at::Tensor* t = plain(p[9]);
    if (!t || !f32_flat(*t, c.B * D, x)) Py_RETURN_NONE;
    c.a.ema_init = fptr(*t);
  }
  at::Tensor out, fin, grad, ws;
  const int dt = p[10] == Py_None ? code(x) : (int)PyLong_AsLong(p[10]);
  if (!out_rows(p[11], dt, &c, &out)) Py_RETURN_NONE;
  const bool want_state = PyObject_IsTrue(p[12]) == 1;
  if (PyErr_Occurred()) return nullptr;
  if (p[13] != Py_None) {
    const at::Tensor* t = plain(p[13]);
    if (!t || t->dim() != 2 || t->size(0) != c.B || t->size(1) != D || !f32_flat(*t, c.B * D, x)) Py_RETURN_NONE;
    fin = *t;
  }
  Ref s_obj;
  void* stream;
  const c10::DeviceGuard guard(x.device());
  if (!stream_of(x, &s_obj, &stream)) return nullptr;
  {
    const NoGil nogil;
    if (!out.defined()) out = empty({c.B, c.S, D}, x, dt == OSM_F32 ? at::kFloat : at::kBFloat16);
    if (!fin.defined() && want_state) fin = empty({c.B, D}, x, at::kFloat);
    if (ttt) grad = empty({c.B, c.H, c.K, c.hd}, x, at::kFloat);
  }
  set_out(&c, out);
  c.a.ema_final = fin.defined() ? fptr(fin) : nullptr;
  const int op = ttt ? OSM_OP_TTT : OSM_OP_FWD;
  const size_t need = lib.workspace_bytes(&c.a, op);
  if (need == 0) Py_RETURN_NONE;   // refused: the Python path says why
  const bool have = get_workspace(p[0], x, s_obj.o, stream, need, op, &ws);
  if (!have) return nullptr;
  int rc;
  {
    const NoGil nogil;
    rc = ttt ? lib.ttt(&c.a, fptr(grad), target, ws.data_ptr(), (size_t)ws.numel(), stream)
             : lib.fwd(&c.a, ws.data_ptr(), (size_t)ws.numel(), stream);
  }
  if (rc != OSM_OK) return fail_rc(rc);
  PyObject* f = Py_None;
  if (want_state)
    f = THPVariable_Wrap(fin);
  else
    Py_INCREF(f);
  if (ttt) return Py_BuildValue("(NNN)", THPVariable_Wrap(out), THPVariable_Wrap(grad), f);
  return Py_BuildValue("(NN)", THPVariable_Wrap(out), f);
}

// backward(<common 9>, out, grad_out, grad_state, need_coeffs, need_init):
// None, or (grad_x, grad_coeffs | None, grad_init | None).
PyObject* run_backward(PyObject* const* p) {
  Common c;
  if (!common(p, &c)) Py_RETURN_NONE;
  const at::Tensor& x = *c.x;
  const int64_t D = c.H * c.hd;
  const at::Tensor *out = plain(p[9]), *go = plain(p[10]);
  if (!out || !go || !(is_f32(*out) || is_bf16(*out)) || out->scalar_type() != go->scalar_type() || !rows(*out, x) ||
      !rows(*go, x))
    Py_RETURN_NONE;
  osm_cheby_bwd_args b{};
  if (p[11] != Py_None) {
    const at::Tensor* t = plain(p[11]);
    if (!t || !f32_flat(*t, c.B * D, x)) Py_RETURN_NONE;
    b.grad_state = fptr(*t);
  }
  const bool need_c = PyObject_IsTrue(p[12]) == 1, need_i = PyObject_IsTrue(p[13]) == 1;
  if (PyErr_Occurred()) return nullptr;
  c.a.out_dtype = code(*out);
  set_out(&c, *out);
  b.grad_out = go->data_ptr();
  b.go_stride_b = go->stride(0);
  b.go_stride_s = go->stride(1);
  Ref s_obj;
  void* stream;
  const c10::DeviceGuard guard(x.device());
  const size_t need = lib.workspace_bytes(&c.a, OSM_OP_BWD);
  if (need == 0) Py_RETURN_NONE;
  if (!stream_of(x, &s_obj, &stream)) return nullptr;
  at::Tensor gx, gc, gi, ws;
  {
    const NoGil nogil;
    gx = empty({c.B, c.S, D}, x, x.scalar_type());
    if (need_c) gc = empty({c.B, c.H, c.K, c.hd}, x, at::kFloat);
    if (need_i) gi = empty({c.B, D}, x, at::kFloat);
  }
  b.grad_x = gx.data_ptr();
  b.gx_stride_b = gx.stride(0);
  b.gx_stride_s = gx.stride(1);
  if (need_c) b.grad_coeffs = fptr(gc);
  if (need_i) b.grad_init = fptr(gi);
  const bool have = get_workspace(p[0], x, s_obj.o, stream, need, OSM_OP_BWD, &ws);
  if (!have) return nullptr;
  int rc;
  {
    const NoGil nogil;
    rc = lib.bwd(&c.a, &b, ws.data_ptr(), (size_t)ws.numel(), stream);
  }
  if (rc != OSM_OK) return fail_rc(rc);
  PyObject *oc = Py_None, *oi = Py_None;
  if (need_c) oc = THPVariable_Wrap(gc); else Py_INCREF(oc);
  if (need_i) oi = THPVariable_Wrap(gi); else Py_INCREF(oi);
  return Py_BuildValue("(NNN)", THPVariable_Wrap(gx), oc, oi);
}

// A momentum: a number, or a one-element fp32 tensor on x's device.
bool momentum(PyObject* o, const at::Tensor& x, float* val, const float** ptr) {
  *val = 0.0f;
  *ptr = nullptr;
  if (THPVariable_Check(o)) {
    const at::Tensor* t = plain(o);
    if (!t || !f32_flat(*t, 1, x)) return false;
    *ptr = fptr(*t);
    return true;
  }
  return as_float(o, val);
}

// [B,H,K,hd] fp32 on x's device with lane stride 1.
bool head_rows(const at::Tensor* t, const at::Tensor& x, int64_t H) {
  return t && t->dim() == 4 && is_f32(*t) && t->device() == x.device() && t->size(0) == x.size(0) && t->size(1) == H &&
         H * t->size(3) == x.size(2) && t->stride(3) == 1;
}

bool batch_vec(PyObject* o, const at::Tensor& x, const float** ptr) {
  *ptr = nullptr;
  if (o == Py_None) return true;
  const at::Tensor* t = plain(o);
  if (!t || !f32_flat(*t, x.size(0), x)) return false;
  *ptr = fptr(*t);
  return true;
}

// v10(x, coeffs, momentum, n_heads, gate, dyn, mu, lut, lion_lambda, ss,
// lr_scale, base_lr, beta1, beta2, weight_decay, chunk, use_lut, save): None,
// or (out, coeffs, momentum) and with save (.., z, coeff_hist).
PyObject* run_v10(PyObject* const* p) {
  const at::Tensor *xp = plain(p[0]), *cp = plain(p[1]), *mp = plain(p[2]);
  if (!xp || !xp->is_cuda() || !(is_f32(*xp) || is_bf16(*xp)) || !rows(*xp, *xp) || xp->size(1) == 0) Py_RETURN_NONE;
  const at::Tensor& x = *xp;
  osm_v10_args a{};
  if (!as_int(p[3], &a.H) || !as_int(p[15], &a.chunk) || a.chunk < 1) Py_RETURN_NONE;
  if (!head_rows(cp, x, a.H) || !head_rows(mp, x, a.H) || mp->sizes() != cp->sizes() || cp->size(2) > 8) Py_RETURN_NONE;
  if (!batch_vec(p[4], x, &a.gate) || !batch_vec(p[5], x, &a.dyn_lambda)) Py_RETURN_NONE;
  if (!momentum(p[6], x, &a.ema_momentum, &a.ema_momentum_dev)) Py_RETURN_NONE;
  if (!as_float(p[11], &a.base_lr) || !as_float(p[12], &a.beta1) || !as_float(p[13], &a.beta2) ||
      !as_float(p[14], &a.weight_decay))
    Py_RETURN_NONE;
  const float** const tables[4] = {&a.lut, &a.lion_lambda, &a.spectral_scale, &a.lr_scale};
  for (int i = 0; i < 4; ++i) *tables[i] = fptr(THPVariable_Unpack(p[7 + i]));   // the module's own tables
  a.abi_version = OSM_ABI_VERSION;
  a.flags = PyObject_IsTrue(p[16]) == 1 ? OSM_V10_USE_LUT : 0;
  const bool save = PyObject_IsTrue(p[17]) == 1;
  if (PyErr_Occurred()) return nullptr;
  a.B = x.size(0);
  a.S = x.size(1);
  a.hd = cp->size(3);
  a.K = cp->size(2);
  const int64_t D = x.size(2), n_chunks = (a.S + a.chunk - 1) / a.chunk;
  Ref s_obj;
  void* stream;
  const c10::DeviceGuard guard(x.device());
  if (!stream_of(x, &s_obj, &stream)) return nullptr;
  at::Tensor out, c_out, m_out, z, hist;
  int rc;
  {
    const NoGil nogil;
    out = empty({a.B, a.S, D}, x, at::kFloat);
    c_out = empty({a.B, a.H, a.K, a.hd}, x, at::kFloat);
    m_out = empty({a.B, a.H, a.K, a.hd}, x, at::kFloat);
    if (save) {
      z = empty({a.B, a.S, D}, x, at::kBFloat16);
      hist = empty({n_chunks, a.B, a.H, a.K, a.hd}, x, at::kFloat);
      a.z_save = z.data_ptr();
      a.z_stride_b = z.stride(0);
      a.z_stride_s = z.stride(1);
      a.coeff_hist = fptr(hist);
    }
    a.x = x.data_ptr();
    a.x_dtype = code(x);
    a.x_stride_b = x.stride(0);
    a.x_stride_s = x.stride(1);
    a.out = fptr(out);
    a.out_stride_b = out.stride(0);
    a.out_stride_s = out.stride(1);
    a.coeffs = fptr(*cp);
    a.c_stride_b = cp->stride(0);
    a.c_stride_h = cp->stride(1);
    a.c_stride_k = cp->stride(2);
    a.momentum = fptr(*mp);
    a.m_stride_b = mp->stride(0);
    a.m_stride_h = mp->stride(1);
    a.m_stride_k = mp->stride(2);
    a.coeffs_out = fptr(c_out);
    a.momentum_out = fptr(m_out);
    rc = lib.v10(&a, stream);
  }
  if (rc != OSM_OK) return fail_rc(rc);
  if (save)
    return Py_BuildValue("(NNNNN)", THPVariable_Wrap(out), THPVariable_Wrap(c_out), THPVariable_Wrap(m_out),
                         THPVariable_Wrap(z), THPVariable_Wrap(hist));
  return Py_BuildValue("(NNN)", THPVariable_Wrap(out), THPVariable_Wrap(c_out), THPVariable_Wrap(m_out));
}

// v10_backward(x, out, z, coeff_hist, grad_out, mu, chunk): None or grad_x.
PyObject* run_v10_backward(PyObject* const* p) {
  const at::Tensor *t[5];
  for (int i = 0; i < 5; ++i)
    if (!(t[i] = plain(p[i]))) Py_RETURN_NONE;
  const at::Tensor &x = *t[0], &out = *t[1], &z = *t[2], &hist = *t[3], &go = *t[4];
  constexpr int64_t kMost = int64_t(1) << 20;   // longer token strides: the Python path copies
  if (!x.is_cuda() || !(is_f32(x) || is_bf16(x)) || !is_f32(out) || !is_bf16(z) || !is_f32(go)) Py_RETURN_NONE;
  for (const at::Tensor* r : {&x, &out, &z, &go})
    if (!rows(*r, x) || r->stride(1) > kMost) Py_RETURN_NONE;
  if (hist.dim() != 5 || !is_f32(hist) || hist.device() != x.device() || !hist.is_contiguous()) Py_RETURN_NONE;
  osm_v10_bwd_args a{};
  if (!momentum(p[5], x, &a.ema_momentum, &a.ema_momentum_dev) || !as_int(p[6], &a.chunk)) Py_RETURN_NONE;
  a.abi_version = OSM_ABI_VERSION;
  a.x_dtype = code(x);
  a.B = x.size(0);
  a.S = x.size(1);
  a.H = hist.size(2);
  a.K = hist.size(3);
  a.hd = hist.size(4);
  if (a.chunk < 1 || a.H * a.hd != x.size(2) || hist.size(1) != a.B || hist.size(0) * a.chunk < a.S) Py_RETURN_NONE;
  Ref s_obj;
  void* stream;
  const c10::DeviceGuard guard(x.device());
  if (!stream_of(x, &s_obj, &stream)) return nullptr;
  at::Tensor gx;
  int rc;
  {
    const NoGil nogil;
    gx = empty(x.sizes(), x, x.scalar_type());
    a.x = x.data_ptr();
    a.x_stride_b = x.stride(0);
    a.x_stride_s = x.stride(1);
    a.grad_out = fptr(go);
    a.go_stride_b = go.stride(0);
    a.go_stride_s = go.stride(1);
    a.out = fptr(out);
    a.out_stride_b = out.stride(0);
    a.out_stride_s = out.stride(1);
    a.z_saved = z.data_ptr();
    a.z_stride_b = z.stride(0);
    a.z_stride_s = z.stride(1);
    a.coeff_hist = fptr(hist);
    a.grad_x = gx.data_ptr();
    a.gx_stride_b = gx.stride(0);
    a.gx_stride_s = gx.stride(1);
    rc = lib.v10_bwd(&a, stream);
  }
  if (rc != OSM_OK) return fail_rc(rc);
  return THPVariable_Wrap(gx);
}

// lut_forward(x, coeffs, n_heads, mu, ema_init, flags, lut, clamp_tile,
// want_x_norm, want_tanh_y): None, or (out, x_norm | None, tanh_y | None, ema_final).
PyObject* run_lut(PyObject* const* p) {
  const at::Tensor *xp = plain(p[0]), *cp = plain(p[1]);
  if (!xp || !xp->is_cuda() || !(is_f32(*xp) || is_bf16(*xp)) || !rows(*xp, *xp)) Py_RETURN_NONE;
  const at::Tensor& x = *xp;
  osm_lut_fwd_args a{};
  if (!as_int(p[2], &a.H) || !as_int(p[7], &a.clamp_tile)) Py_RETURN_NONE;
  if (!head_rows(cp, x, a.H) || cp->size(2) < 1 || cp->size(2) > 8 || !as_float(p[3], &a.ema_momentum)) Py_RETURN_NONE;
  a.B = x.size(0);
  a.S = x.size(1);
  a.hd = cp->size(3);
  a.K = cp->size(2);
  const int64_t D = x.size(2);
  if (p[4] != Py_None) {
    const at::Tensor* t = plain(p[4]);
    if (!t || t->dim() != 2 || t->size(0) != a.B || t->size(1) != D || !f32_flat(*t, a.B * D, x)) Py_RETURN_NONE;
    a.ema_init = fptr(*t);
    a.init_stride_b = t->stride(0);
  }
  a.flags = (int32_t)PyLong_AsLong(p[5]);
  if (a.flags & OSM_V10_USE_LUT) a.lut = fptr(THPVariable_Unpack(p[6]));   // the module's own table
  const bool want_n = PyObject_IsTrue(p[8]) == 1, want_y = PyObject_IsTrue(p[9]) == 1;
  if (PyErr_Occurred()) return nullptr;
  a.abi_version = OSM_ABI_VERSION;
  a.x = x.data_ptr();
  a.x_dtype = code(x);
  a.x_stride_b = x.stride(0);
  a.x_stride_s = x.stride(1);
  a.coeffs = fptr(*cp);
  a.c_stride_b = cp->stride(0);
  a.c_stride_h = cp->stride(1);
  a.c_stride_k = cp->stride(2);
  Ref s_obj;
  void* stream;
  const c10::DeviceGuard guard(x.device());
  if (!stream_of(x, &s_obj, &stream)) return nullptr;
  at::Tensor out, xn, ty, fin, ws;
  {
    const NoGil nogil;
    out = empty({a.B, a.S, D}, x, at::kFloat);
    if (want_n) xn = empty({a.B, a.S, D}, x, at::kFloat);
    if (want_y) ty = empty({a.B, a.S, D}, x, at::kFloat);
    fin = empty({a.B, D}, x, at::kFloat);
  }
  a.out = fptr(out);
  a.out_stride_b = out.stride(0);
  a.out_stride_s = out.stride(1);
  if (want_n) {
    a.x_norm = fptr(xn);
    a.xn_stride_b = xn.stride(0);
    a.xn_stride_s = xn.stride(1);
  }
  if (want_y) {
    a.tanh_y = fptr(ty);
    a.ty_stride_b = ty.stride(0);
    a.ty_stride_s = ty.stride(1);
  }
  a.ema_final = fptr(fin);
  a.final_stride_b = fin.stride(0);
  const size_t need = lib.lut_bytes(&a);
  if (need && !get_workspace(p[0], x, s_obj.o, stream, need, kOpLut, &ws)) return nullptr;
  int rc;
  {
    const NoGil nogil;
    rc = lib.lut_ws(&a, need ? ws.data_ptr() : nullptr, need ? (size_t)ws.numel() : 0, stream);
  }
  if (rc != OSM_OK) return fail_rc(rc);
  PyObject *on = Py_None, *oy = Py_None;
  if (want_n) on = THPVariable_Wrap(xn); else Py_INCREF(on);
  if (want_y) oy = THPVariable_Wrap(ty); else Py_INCREF(oy);
  return Py_BuildValue("(NNNN)", THPVariable_Wrap(out), on, oy, THPVariable_Wrap(fin));
}

// engine(x, norm_weight, eps, w1, b1, w2, b2, ema_base, tokens_seen): None, or
// (x_normed, gate, mu).
PyObject* run_engine(PyObject* const* p) {
  const at::Tensor* const xp = plain(p[0]);
  if (!xp || !xp->is_cuda() || !is_f32(*xp) || !rows(*xp, *xp) || xp->numel() == 0) Py_RETURN_NONE;
  const at::Tensor& x = *xp;
  const int64_t D = x.size(2), sizes[6] = {D, D / 4 * D, D / 4, D / 4, 1, 1};
  const int at[6] = {1, 3, 4, 5, 6, 7};   // norm_weight, w1, b1, w2, b2, ema_base
  for (int i = 0; i < 6; ++i) {
    const at::Tensor* t = plain(p[at[i]]);
    if (!t || !f32_flat(*t, sizes[i], x)) Py_RETURN_NONE;
  }
  const at::Tensor* seen = plain(p[8]);
  if (!seen || seen->scalar_type() != at::kLong || seen->numel() != 1 || seen->device() != x.device()) Py_RETURN_NONE;
  auto ptr = [&](int i) { return fptr(THPVariable_Unpack(p[i])); };
  osm_engine_args a{};
  if (!as_float(p[2], &a.eps)) Py_RETURN_NONE;
  a.abi_version = OSM_ABI_VERSION;
  a.B = x.size(0);
  a.S = x.size(1);
  a.D = D;
  a.x = fptr(x);
  a.x_stride_b = x.stride(0);
  a.x_stride_s = x.stride(1);
  a.norm_weight = ptr(1);
  a.w1 = ptr(3);
  a.b1 = ptr(4);
  a.w2 = ptr(5);
  a.b2 = ptr(6);
  a.ema_base = ptr(7);
  a.tokens_seen = static_cast<int64_t*>(seen->data_ptr());
  Ref s_obj;
  void* stream;
  const c10::DeviceGuard guard(x.device());
  if (!stream_of(x, &s_obj, &stream)) return nullptr;
  at::Tensor xn, scratch, gate, mu;
  int rc;
  {
    const NoGil nogil;
    xn = empty({a.B, a.S, a.D}, x, at::kFloat);
    scratch = empty({(int64_t)(lib.engine_bytes(a.B, a.S, a.D) / 4)}, x, at::kFloat);
    gate = empty({a.B, 1}, x, at::kFloat);
    mu = empty({}, x, at::kFloat);
    a.x_normed = fptr(xn);
    a.scratch = fptr(scratch);
    a.gate = fptr(gate);
    a.ema_momentum = fptr(mu);
    rc = lib.engine(&a, stream);
  }
  if (rc != OSM_OK) return fail_rc(rc);
  return Py_BuildValue("(NNN)", THPVariable_Wrap(xn), THPVariable_Wrap(gate), THPVariable_Wrap(mu));
}

// ---- gated delta rule, layer norm, gradient clipping (orthossm_amd/delta.py,
// norm.py, grad_clip.py): as above, None for what is not in the kernels' form.
// Their scratch memory is a plain allocation: nothing in it outlives the call.

PyObject* wrap_or_none(const at::Tensor& t) {
  if (t.defined()) return THPVariable_Wrap(t);
  Py_RETURN_NONE;
}

at::Tensor scratch(size_t bytes, const at::Tensor& like) { return empty({(int64_t)bytes}, like, at::kByte); }

osm_rows rows_of(const at::Tensor& t) { return {t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)}; }

// Tokens' rows as the kernels address them.
bool token_rows(const at::Tensor& t, int64_t dim) {
  const int64_t s = t.size(1) > 1 ? t.stride(1) : dim;
  return t.stride(0) >= 0 && t.stride(2) >= 0 && s >= dim && s <= OSM_DELTA_MAX_STRIDE && (dim == 1 || t.stride(3) == 1);
}

// A scale: a number, or None for 1/sqrt(dk).
bool as_scale(PyObject* o, int64_t dk, float* v) {
  if (o == Py_None) {
    *v = (float)(1.0 / std::sqrt((double)dk));
    return true;
  }
  return as_float(o, v);
}

// Whether t is a dual number of forward-mode differentiation, which the operators
// have no derivative for: the Python functions' autograd functions refuse it.
bool has_tangent(const at::Tensor& t) { return t._fw_grad(0).defined(); }

// Tells autograd that a launch wrote into t: a graph that saved it refuses its
// backward.  (Inference tensors have no version, and no graph saves them.)
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

std::optional<at::Tensor> optional_tensor(PyObject* o) {
  return o == Py_None ? std::nullopt : std::optional<at::Tensor>(*plain(o));
}

// ---- in the autograd engine's threads, which run without the interpreter's lock ----

// The interpreter's lock, for a scope.
struct Gil {
  PyGILState_STATE s = PyGILState_Ensure();
  ~Gil() { PyGILState_Release(s); }
};

[[noreturn]] void throw_python() {
  python_error e;
  e.persist();
  throw e;
}

// The stream that the engine has made current: the forward's.
void* engine_stream(const at::Tensor& x) {
  const Gil gil;
  Ref obj;
  void* stream;
  if (!stream_of(x, &obj, &stream)) throw_python();
  return stream;
}

// The Python error of a status code, thrown.
void throw_rc(int rc) {
  if (rc == OSM_OK) return;
  const Gil gil;
  fail_rc(rc);
  throw_python();
}

// Gradients that are themselves part of a graph (create_graph): the identity,
// with a backward that refuses.
struct Once : torch::autograd::Function<Once> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext*, at::TensorList grads, at::TensorList) {
    torch::autograd::variable_list res;
    for (const at::Tensor& t : grads) res.push_back(t.view_as(t));
    return res;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext*, torch::autograd::variable_list) {
    TORCH_CHECK(false, "trying to differentiate twice a function that can be differentiated once only");
  }
};
torch::autograd::variable_list once(torch::autograd::variable_list res, const torch::autograd::variable_list& of) {
  if (!at::GradMode::is_enabled()) return res;
  torch::autograd::variable_list grads, from;
  for (const at::Tensor& t : res)
    if (t.defined()) grads.push_back(t);
  for (const at::Tensor& t : of)
    if (t.defined()) from.push_back(t);
  const torch::autograd::variable_list refusing = Once::apply(at::TensorList(grads), at::TensorList(from));
  size_t i = 0;
  for (at::Tensor& t : res)
    if (t.defined()) t = refusing[i++];
  return res;
}

// A hook on saved tensors can give back anything, which the kernels would read as
// what was saved.
constexpr const char* kAnotherForm = "a saved tensor came back in another form: ";

struct Delta {
  const at::Tensor* t[5];        // q, k, v, g, beta
  osm_delta_args a{};
};

bool delta_tensors(Delta* d) {
  for (int i = 0; i < 5; ++i)
    if (!d->t[i]->is_cuda() || d->t[i]->dim() != (i < 3 ? 4 : 3)) return false;
  const at::Tensor &q = *d->t[0], &k = *d->t[1], &v = *d->t[2];
  if (!(is_f32(q) || is_bf16(q)) || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type()) return false;
  osm_delta_args& a = d->a;
  a.abi_version = OSM_ABI_VERSION;
  a.dtype = code(q);
  a.B = q.size(0);
  a.S = q.size(1);
  a.Hk = q.size(2);
  a.dk = q.size(3);
  a.H = v.size(2);
  a.dv = v.size(3);
  if (k.sizes() != q.sizes() || v.size(0) != a.B || v.size(1) != a.S || a.Hk < 1 || a.H < 1 || a.H % a.Hk || a.dk < 1 ||
      a.dk > OSM_DELTA_MAX_DK || a.dv < 1)
    return false;
  for (int i = 0; i < 5; ++i) {
    const at::Tensor& t = *d->t[i];
    if (t.device() != q.device()) return false;
    if (i < 3 ? !token_rows(t, t.size(3))
              : !is_f32(t) || t.size(0) != a.B || t.size(1) != a.S || t.size(2) != a.H || t.stride(0) < 0 ||
                    t.stride(2) < 0 || (a.S > 1 && (t.stride(1) < 0 || t.stride(1) > OSM_DELTA_MAX_STRIDE)))
      return false;
  }
  a.q = rows_of(q);
  a.k = rows_of(k);
  a.v = rows_of(v);
  a.g = rows_of(*d->t[3]);
  a.beta = rows_of(*d->t[4]);
  return true;
}

bool lengths_form(const at::Tensor& t, const Delta& d) {
  return t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == d.a.B && t.is_contiguous() &&
         t.device() == d.t[0]->device();
}

// What the forward saved of these inputs for the backward.
bool saved_form(const at::Tensor& t, const Delta& d) {
  return t.scalar_type() == at::kByte && (size_t)t.numel() == lib.delta_saved(&d.a) && t.is_contiguous() &&
         t.device() == d.t[0]->device();
}

// args: q, k, v, g, beta, scale, lengths.
bool delta_common(PyObject* const* p, Delta* d) {
  for (int i = 0; i < 5; ++i)
    if (!(d->t[i] = plain(p[i]))) return false;
  if (!delta_tensors(d)) return false;
  osm_delta_args& a = d->a;
  if (!as_scale(p[5], a.dk, &a.scale)) return false;
  if (p[6] != Py_None) {
    const at::Tensor* t = plain(p[6]);
    if (!t || !lengths_form(*t, *d)) return false;
    a.lengths = static_cast<const int32_t*>(t->data_ptr());
  }
  return true;
}

// A state [B,H,dk,dv] fp32 contiguous, or None; false for another.
bool state_ptr(PyObject* o, const Delta& d, float** out) {
  *out = nullptr;
  if (o == Py_None) return true;
  const at::Tensor* t = plain(o);
  if (!t || t->dim() != 4 || t->size(0) != d.a.B || t->size(1) != d.a.H || t->size(2) != d.a.dk || t->size(3) != d.a.dv ||
      !f32_flat(*t, t->numel(), *d.t[0]))
    return false;
  *out = fptr(*t);
  return true;
}

// A gradient of the output as the kernels read it.
bool delta_grad_form(const at::Tensor& go, const at::Tensor& v) {
  return go.dim() == 4 && go.sizes() == v.sizes() && go.scalar_type() == v.scalar_type() && go.device() == v.device() &&
         token_rows(go, v.size(3));
}

// The forward into new tensors, those of `fin` and `saved` where wanted.
int delta_forward(Delta& d, bool want_state, bool save, void* stream, at::Tensor* out, at::Tensor* fin, at::Tensor* saved) {
  const at::Tensor& q = *d.t[0];
  osm_delta_args& a = d.a;
  *out = empty({a.B, a.S, a.H, a.dv}, q, q.scalar_type());
  a.out = rows_of(*out);
  if (want_state) {
    *fin = empty({a.B, a.H, a.dk, a.dv}, q, at::kFloat);
    a.state_out = fptr(*fin);
  }
  if (save) {
    *saved = scratch(lib.delta_saved(&a), q);
    a.saved = saved->data_ptr();
  }
  const at::Tensor ws = scratch(lib.delta_bytes(&a), q);
  return lib.delta_fwd(&a, ws.data_ptr(), (size_t)ws.numel(), stream);
}

// The six gradients into new tensors, that of the first state where needed.
int delta_backward(Delta& d, const at::Tensor& go, float* grad_state, bool need_init, void* stream, at::Tensor* gr) {
  const at::Tensor& q = *d.t[0];
  osm_delta_args& a = d.a;
  osm_delta_bwd_args b{};
  b.grad_out = rows_of(go);
  b.grad_state = grad_state;
  for (int i = 0; i < 5; ++i) gr[i] = empty(d.t[i]->sizes(), q, d.t[i]->scalar_type());
  b.grad_q = rows_of(gr[0]);
  b.grad_k = rows_of(gr[1]);
  b.grad_v = rows_of(gr[2]);
  b.grad_g = rows_of(gr[3]);
  b.grad_beta = rows_of(gr[4]);
  if (need_init) {
    gr[5] = empty({a.B, a.H, a.dk, a.dv}, q, at::kFloat);
    b.grad_init = fptr(gr[5]);
  }
  const at::Tensor ws = scratch(lib.delta_bwd_bytes(&a), q);
  return lib.delta_bwd(&a, &b, ws.data_ptr(), (size_t)ws.numel(), stream);
}

// delta_forward(<common 7>, state_init, want_state, save): None, or (out, state | None, saved | None).
PyObject* run_delta_forward(PyObject* const* p) {
  Delta d;
  float* init;
  if (!delta_common(p, &d) || !state_ptr(p[7], d, &init)) Py_RETURN_NONE;
  const bool want_state = PyObject_IsTrue(p[8]) == 1, save = PyObject_IsTrue(p[9]) == 1;
  if (PyErr_Occurred()) return nullptr;
  d.a.state_init = init;
  Ref s_obj;
  void* stream;
  const c10::DeviceGuard guard(d.t[0]->device());
  if (!stream_of(*d.t[0], &s_obj, &stream)) return nullptr;
  at::Tensor out, fin, saved;
  int rc;
  {
    const NoGil nogil;
    rc = delta_forward(d, want_state, save, stream, &out, &fin, &saved);
  }
  if (rc != OSM_OK) return fail_rc(rc);
  return Py_BuildValue("(NNN)", THPVariable_Wrap(out), wrap_or_none(fin), wrap_or_none(saved));
}

// delta_backward(<common 7>, saved, grad_out, grad_state, need_init): None, or the six gradients.
PyObject* run_delta_backward(PyObject* const* p) {
  Delta d;
  float* gs;
  if (!delta_common(p, &d) || !state_ptr(p[9], d, &gs)) Py_RETURN_NONE;
  const at::Tensor &q = *d.t[0], &v = *d.t[2];
  const at::Tensor *saved = plain(p[7]), *go = plain(p[8]);
  if (!saved || !saved_form(*saved, d) || !go || !delta_grad_form(*go, v)) Py_RETURN_NONE;
  const bool need_init = PyObject_IsTrue(p[10]) == 1;
  if (PyErr_Occurred()) return nullptr;
  d.a.saved = saved->data_ptr();
  Ref s_obj;
  void* stream;
  const c10::DeviceGuard guard(q.device());
  if (!stream_of(q, &s_obj, &stream)) return nullptr;
  at::Tensor gr[6];
  int rc;
  {
    const NoGil nogil;
    rc = delta_backward(d, *go, gs, need_init, stream, gr);
  }
  if (rc != OSM_OK) return fail_rc(rc);
  return Py_BuildValue("(NNNNNN)", THPVariable_Wrap(gr[0]), THPVariable_Wrap(gr[1]), THPVariable_Wrap(gr[2]),
                       THPVariable_Wrap(gr[3]), THPVariable_Wrap(gr[4]), wrap_or_none(gr[5]));
}

// The differentiable form: what the Python module's autograd function keeps and
// gives, without the interpreter between the engine and the launches.
struct DeltaCall {
  Delta* d;
  void* stream;
  int rc;
};
struct DeltaGrad : torch::autograd::Function<DeltaGrad> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& q,
                                                const at::Tensor& k, const at::Tensor& v, const at::Tensor& g,
                                                const at::Tensor& beta, const std::optional<at::Tensor>& init,
                                                const std::optional<at::Tensor>& lengths, DeltaCall* c) {
    ctx->set_materialize_grads(false);   // an unused output's gradient stays undefined
    at::Tensor out, fin, saved;
    c->rc = delta_forward(*c->d, true, true, c->stream, &out, &fin, &saved);
    ctx->save_for_backward({q, k, v, g, beta, lengths ? *lengths : at::Tensor(), saved});
    int64_t need = 0;
    const at::Tensor* const t[6] = {&q, &k, &v, &g, &beta, init ? &*init : nullptr};
    for (int i = 0; i < 6; ++i) need |= (int64_t)(t[i] && t[i]->requires_grad()) << i;
    ctx->saved_data["need"] = need;
    ctx->saved_data["scale"] = (double)c->d->a.scale;
    return {out, fin};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const auto t = ctx->get_saved_variables();
    const int64_t need = ctx->saved_data["need"].toInt();
    at::Tensor gr[6];
    {
      const at::NoGradGuard no_grad;
      Delta d;
      for (int i = 0; i < 5; ++i) d.t[i] = &t[i];
      const bool inputs = delta_tensors(&d);
      TORCH_CHECK(inputs && (!t[5].defined() || lengths_form(t[5], d)) && saved_form(t[6], d), kAnotherForm, "gated_delta");
      d.a.scale = (float)ctx->saved_data["scale"].toDouble();
      if (t[5].defined()) d.a.lengths = static_cast<const int32_t*>(t[5].data_ptr());
      d.a.saved = t[6].data_ptr();
      const c10::DeviceGuard guard(t[0].device());
      at::Tensor go = grads[0].defined() ? grads[0] : at::zeros_like(t[2]);
      if (!delta_grad_form(go, t[2])) go = go.to(t[2].options()).contiguous();
      const at::Tensor gs = grads[1].defined() ? grads[1].to(at::kFloat).contiguous() : at::Tensor();
      TORCH_CHECK(delta_grad_form(go, t[2]) && (!gs.defined() || f32_flat(gs, d.a.B * d.a.H * d.a.dk * d.a.dv, t[0])),
                  kAnotherForm, "gated_delta");
      throw_rc(delta_backward(d, go, gs.defined() ? fptr(gs) : nullptr, need >> 5 & 1, engine_stream(t[0]), gr));
    }
    torch::autograd::variable_list res(8);
    for (int i = 0; i < 6; ++i)
      if (need >> i & 1) res[i] = gr[i];
    return once(std::move(res), {grads[0], grads[1], t[0], t[1], t[2], t[3], t[4]});
  }
};

// gated_delta(<common 7>, state_init, return_state): None, or (out, state | None) with their gradient's function.
PyObject* run_gated_delta(PyObject* const* p) {
  Delta d;
  float* init;
  if (!delta_common(p, &d) || !state_ptr(p[7], d, &init)) Py_RETURN_NONE;
  const std::optional<at::Tensor> first = optional_tensor(p[7]), lengths = optional_tensor(p[6]);
  bool grad = first && first->requires_grad(), dual = first && has_tangent(*first);
  for (int i = 0; i < 5; ++i) {
    grad = grad || d.t[i]->requires_grad();
    dual = dual || has_tangent(*d.t[i]);
  }
  if (dual) Py_RETURN_NONE;
  const bool want_state = PyObject_IsTrue(p[8]) == 1;
  if (PyErr_Occurred()) return nullptr;
  d.a.state_init = init;
  Ref s_obj;
  void* stream;
  const c10::DeviceGuard guard(d.t[0]->device());
  if (!stream_of(*d.t[0], &s_obj, &stream)) return nullptr;
  at::Tensor out, fin, saved;
  int rc;
  {
    const NoGil nogil;
    if (grad && at::GradMode::is_enabled()) {
      DeltaCall c{&d, stream, OSM_OK};
      const auto res = DeltaGrad::apply(*d.t[0], *d.t[1], *d.t[2], *d.t[3], *d.t[4], first, lengths, &c);
      rc = c.rc;
      out = res[0];
      if (want_state) fin = res[1];
    } else {
      rc = delta_forward(d, want_state, false, stream, &out, &fin, &saved);
    }
  }
  if (rc != OSM_OK) return fail_rc(rc);
  return Py_BuildValue("(NN)", THPVariable_Wrap(out), wrap_or_none(fin));
}

// delta_step(q, k, v, g, beta, state, scale, slots): None, or out.
PyObject* run_delta_step(PyObject* const* p) {
  const at::Tensor* t[6];
  for (int i = 0; i < 6; ++i) {
    t[i] = plain(p[i]);
    if (!t[i] || !t[i]->is_cuda() || t[i]->device() != t[0]->device()) Py_RETURN_NONE;
  }
  const at::Tensor &q = *t[0], &k = *t[1], &v = *t[2], &state = *t[5];
  if (q.dim() != 3 || v.dim() != 3 || k.sizes() != q.sizes() || !(is_f32(q) || is_bf16(q)) ||
      k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type())
    Py_RETURN_NONE;
  osm_delta_step_args a{};
  a.abi_version = OSM_ABI_VERSION;
  a.dtype = code(q);
  a.B = q.size(0);
  a.Hk = q.size(1);
  a.dk = q.size(2);
  a.H = v.size(1);
  a.dv = v.size(2);
  if (v.size(0) != a.B || a.Hk < 1 || a.H < 1 || a.H % a.Hk || a.dk < 1 || a.dk > OSM_DELTA_MAX_DK || a.dv < 1)
    Py_RETURN_NONE;
  for (int i = 0; i < 5; ++i) {
    const at::Tensor& x = *t[i];
    if (x.stride(0) < 0 || x.stride(1) < 0) Py_RETURN_NONE;
    if (i < 3 ? x.stride(2) != 1 && x.size(2) != 1 : x.dim() != 2 || !is_f32(x) || x.size(0) != a.B || x.size(1) != a.H)
      Py_RETURN_NONE;
    osm_rows* const r = i == 0 ? &a.q : i == 1 ? &a.k : i == 2 ? &a.v : i == 3 ? &a.g : &a.beta;
    *r = {x.data_ptr(), x.stride(0), 0, x.stride(1)};
  }
  if (state.dim() != 4 || !is_f32(state) || state.requires_grad() || state.size(1) != a.H || state.size(2) != a.dk ||
      state.size(3) != a.dv || state.stride(3) != 1 || state.stride(2) != a.dv || state.stride(1) != a.dk * a.dv ||
      state.stride(0) < a.H * a.dk * a.dv)
    Py_RETURN_NONE;
  a.state = fptr(state);
  a.state_stride = state.stride(0);
  a.n_slots = state.size(0);
  if (!as_scale(p[6], a.dk, &a.scale)) Py_RETURN_NONE;
  if (p[7] == Py_None) {
    if (a.n_slots < a.B) Py_RETURN_NONE;
  } else {
    const at::Tensor* s = plain(p[7]);
    if (!s || s->scalar_type() != at::kLong || s->dim() != 1 || s->size(0) != a.B || !s->is_contiguous() ||
        s->device() != q.device())
      Py_RETURN_NONE;
    a.slots = static_cast<const int64_t*>(s->data_ptr());
  }
  Ref s_obj;
  void* stream;
  const c10::DeviceGuard guard(q.device());
  if (!stream_of(q, &s_obj, &stream)) return nullptr;
  at::Tensor out;
  int rc;
  {
    const NoGil nogil;
    out = empty({a.B, a.H, a.dv}, q, q.scalar_type());
    a.out = {out.data_ptr(), out.stride(0), 0, out.stride(1)};
    rc = lib.delta_step(&a, stream);
  }
  if (rc != OSM_OK) return fail_rc(rc);
  written(state);
  return THPVariable_Wrap(out);
}

// x [.., D] whose rows are D contiguous elements, one after the other.
bool norm_rows(const at::Tensor* x) {
  return x && x->is_cuda() && (is_f32(*x) || is_bf16(*x)) && x->dim() >= 1 && x->is_contiguous() &&
         x->size(x->dim() - 1) >= 1;
}

// A parameter [D] fp32, or None; false for another.
bool norm_param(PyObject* o, int64_t D, const at::Tensor& x, const float** out) {
  *out = nullptr;
  if (o == Py_None) return true;
  const at::Tensor* t = plain(o);
  if (!f32_vec(t, D, x)) return false;
  *out = fptr(*t);
  return true;
}

void norm_args(const at::Tensor& x, osm_norm_args* a) {
  a->abi_version = OSM_ABI_VERSION;
  a->dtype = code(x);
  a->D = x.size(x.dim() - 1);
  a->rows = x.numel() / a->D;
  a->x = x.data_ptr();
  a->x_stride = a->D;
}

// A gradient of the output as the kernels read it.
bool norm_grad_form(const at::Tensor& gy, const at::Tensor& x) {
  return norm_rows(&gy) && gy.sizes() == x.sizes() && gy.scalar_type() == x.scalar_type() && gy.device() == x.device();
}

// The forward into new tensors, those of the statistics where wanted.
int norm_forward(osm_norm_args& a, const at::Tensor& x, bool stats, void* stream, at::Tensor* y, at::Tensor* mean,
                 at::Tensor* rstd) {
  *y = empty(x.sizes(), x, x.scalar_type());
  a.y = y->data_ptr();
  a.y_stride = a.D;
  if (stats) {
    const at::IntArrayRef lead = x.sizes().slice(0, x.dim() - 1);
    *mean = empty(lead, x, at::kFloat);
    *rstd = empty(lead, x, at::kFloat);
    a.mean = fptr(*mean);
    a.rstd = fptr(*rstd);
  }
  return lib.norm_fwd(&a, stream);
}

// The gradients that are needed, to x, weight and bias, into new tensors.
int norm_backward(const osm_norm_args& a, const at::Tensor& x, const at::Tensor& gy, const bool* need, void* stream,
                  at::Tensor* gr) {
  osm_norm_bwd_args b{};
  b.grad_y = gy.data_ptr();
  b.grad_y_stride = a.D;
  if (need[0]) {
    gr[0] = empty(x.sizes(), x, x.scalar_type());
    b.grad_x = gr[0].data_ptr();
    b.grad_x_stride = a.D;
  }
  if (need[1]) {
    gr[1] = empty({a.D}, x, at::kFloat);
    b.grad_weight = fptr(gr[1]);
  }
  if (need[2]) {
    gr[2] = empty({a.D}, x, at::kFloat);
    b.grad_bias = fptr(gr[2]);
  }
  const at::Tensor ws = scratch(lib.norm_bwd_bytes(&a), x);
  return lib.norm_bwd(&a, &b, ws.data_ptr(), (size_t)ws.numel(), stream);
}

// norm_forward(x, weight, bias, eps, stats): None, or (y, mean | None, rstd | None).
PyObject* run_norm_forward(PyObject* const* p) {
  const at::Tensor* const xp = plain(p[0]);
  if (!norm_rows(xp)) Py_RETURN_NONE;
  const at::Tensor& x = *xp;
  osm_norm_args a{};
  norm_args(x, &a);
  if (!norm_param(p[1], a.D, x, &a.weight) || !norm_param(p[2], a.D, x, &a.bias) || !as_float(p[3], &a.eps)) Py_RETURN_NONE;
  const bool stats = PyObject_IsTrue(p[4]) == 1;
  if (PyErr_Occurred()) return nullptr;
  Ref s_obj;
  void* stream;
  const c10::DeviceGuard guard(x.device());
  if (!stream_of(x, &s_obj, &stream)) return nullptr;
  at::Tensor y, mean, rstd;
  int rc;
  {
    const NoGil nogil;
    rc = norm_forward(a, x, stats, stream, &y, &mean, &rstd);
  }
  if (rc != OSM_OK) return fail_rc(rc);
  return Py_BuildValue("(NNN)", THPVariable_Wrap(y), wrap_or_none(mean), wrap_or_none(rstd));
}

// norm_backward(grad_y, x, mean, rstd, weight, need_x, need_weight, need_bias): None, or
// (grad_x | None, grad_weight | None, grad_bias | None).
PyObject* run_norm_backward(PyObject* const* p) {
  const at::Tensor *const gyp = plain(p[0]), *const xp = plain(p[1]), *const mp = plain(p[2]), *const rp = plain(p[3]);
  if (!norm_rows(xp) || !gyp || !norm_grad_form(*gyp, *xp) || !mp || !rp) Py_RETURN_NONE;
  const at::Tensor& x = *xp;
  osm_norm_args a{};
  norm_args(x, &a);
  if (!f32_flat(*mp, a.rows, x) || !f32_flat(*rp, a.rows, x) || mp->dim() != x.dim() - 1 || rp->dim() != x.dim() - 1 ||
      !norm_param(p[4], a.D, x, &a.weight))
    Py_RETURN_NONE;
  a.mean = fptr(*mp);
  a.rstd = fptr(*rp);
  bool need[3];
  for (int i = 0; i < 3; ++i) need[i] = PyObject_IsTrue(p[5 + i]) == 1;
  if (PyErr_Occurred()) return nullptr;
  Ref s_obj;
  void* stream;
  const c10::DeviceGuard guard(x.device());
  if (!stream_of(x, &s_obj, &stream)) return nullptr;
  at::Tensor gr[3];
  int rc;
  {
    const NoGil nogil;
    rc = norm_backward(a, x, *gyp, need, stream, gr);
  }
  if (rc != OSM_OK) return fail_rc(rc);
  return Py_BuildValue("(NNN)", wrap_or_none(gr[0]), wrap_or_none(gr[1]), wrap_or_none(gr[2]));
}

// The differentiable form (see DeltaGrad).
struct NormCall {
  osm_norm_args* a;
  void* stream;
  int rc;
};
struct NormGrad : torch::autograd::Function<NormGrad> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x,
                            const std::optional<at::Tensor>& weight, const std::optional<at::Tensor>& bias, NormCall* c) {
    at::Tensor y, mean, rstd;
    c->rc = norm_forward(*c->a, x, true, c->stream, &y, &mean, &rstd);
    ctx->save_for_backward({x, mean, rstd, weight ? *weight : at::Tensor()});
    ctx->saved_data["need"] = (int64_t)(x.requires_grad() | (weight && weight->requires_grad()) << 1 |
                                        (bias && bias->requires_grad()) << 2);
    return y;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const auto t = ctx->get_saved_variables();
    const int64_t bits = ctx->saved_data["need"].toInt();
    const bool need[3] = {(bits & 1) != 0, (bits & 2) != 0, (bits & 4) != 0};
    torch::autograd::variable_list res(4);
    {
      const at::NoGradGuard no_grad;
      const at::Tensor& x = t[0];
      TORCH_CHECK(norm_rows(&x), kAnotherForm, "layer_norm");
      osm_norm_args a{};
      norm_args(x, &a);
      TORCH_CHECK(f32_flat(t[1], a.rows, x) && f32_flat(t[2], a.rows, x) && (!t[3].defined() || f32_vec(&t[3], a.D, x)),
                  kAnotherForm, "layer_norm");
      a.mean = fptr(t[1]);
      a.rstd = fptr(t[2]);
      if (t[3].defined()) a.weight = fptr(t[3]);
      const c10::DeviceGuard guard(x.device());
      const at::Tensor gy = norm_grad_form(grads[0], x) ? grads[0] : grads[0].to(x.options()).contiguous();
      TORCH_CHECK(norm_grad_form(gy, x), kAnotherForm, "layer_norm");
      throw_rc(norm_backward(a, x, gy, need, engine_stream(x), res.data()));
    }
    return once(std::move(res), {grads[0], t[0], t[3]});
  }
};

// layer_norm(x, weight, bias, eps): None, or y with its gradient's function.
PyObject* run_layer_norm(PyObject* const* p) {
  const at::Tensor* const xp = plain(p[0]);
  if (!norm_rows(xp)) Py_RETURN_NONE;
  const at::Tensor& x = *xp;
  osm_norm_args a{};
  norm_args(x, &a);
  if (!norm_param(p[1], a.D, x, &a.weight) || !norm_param(p[2], a.D, x, &a.bias) || !as_float(p[3], &a.eps)) Py_RETURN_NONE;
  const std::optional<at::Tensor> weight = optional_tensor(p[1]), bias = optional_tensor(p[2]);
  if (has_tangent(x) || (weight && has_tangent(*weight)) || (bias && has_tangent(*bias))) Py_RETURN_NONE;
  Ref s_obj;
  void* stream;
  const c10::DeviceGuard guard(x.device());
  if (!stream_of(x, &s_obj, &stream)) return nullptr;
  const bool grad = x.requires_grad() || (weight && weight->requires_grad()) || (bias && bias->requires_grad());
  at::Tensor y, mean, rstd;
  int rc;
  {
    const NoGil nogil;
    if (grad && at::GradMode::is_enabled()) {
      NormCall c{&a, stream, OSM_OK};
      y = NormGrad::apply(x, weight, bias, &c);
      rc = c.rc;
    } else {
      rc = norm_forward(a, x, false, stream, &y, &mean, &rstd);
    }
  }
  if (rc != OSM_OK) return fail_rc(rc);
  return THPVariable_Wrap(y);
}

// clip(tensors, max_norm, eps, scale): None, or the norm.  tensors: a list or tuple.
PyObject* run_clip(PyObject* const* p) {
  if (!PyList_Check(p[0]) && !PyTuple_Check(p[0])) Py_RETURN_NONE;
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(p[0]);
  if (n == 0) Py_RETURN_NONE;
  const double max_norm = PyFloat_AsDouble(p[1]), eps = PyFloat_AsDouble(p[2]);
  const bool scale = PyObject_IsTrue(p[3]) == 1;
  if (PyErr_Occurred()) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  std::vector<void*> ptr(n);
  std::vector<int64_t> size(n);
  std::vector<int32_t> dtype(n);
  std::vector<at::Tensor> held;   // (the list may change while the lock is released)
  held.reserve(n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    const at::Tensor* const t = plain(PySequence_Fast_GET_ITEM(p[0], i));
    if (!t || !t->is_cuda() || !(is_f32(*t) || is_bf16(*t)) || !t->is_contiguous() || (scale && t->requires_grad()))
      Py_RETURN_NONE;
    if (i > 0 && t->device() != held[0].device()) Py_RETURN_NONE;
    held.push_back(*t);
    ptr[i] = t->data_ptr();
    size[i] = t->numel();
    dtype[i] = code(*t);
  }
  osm_clip_args a{};
  a.abi_version = OSM_ABI_VERSION;
  a.flags = scale ? OSM_CLIP_SCALE : 0;
  a.count = n;
  a.tensors = ptr.data();
  a.sizes = size.data();
  a.dtypes = dtype.data();
  a.max_norm = max_norm;
  a.eps = eps;
  Ref s_obj;
  void* stream;
  const at::Tensor& first = held[0];
  const c10::DeviceGuard guard(first.device());
  if (!stream_of(first, &s_obj, &stream)) return nullptr;
  at::Tensor norm, ws;
  int rc;
  {
    const NoGil nogil;
    norm = empty({}, first, at::kFloat);
    a.norm = fptr(norm);
    ws = scratch(lib.clip_bytes(&a), first);
    rc = lib.clip(&a, ws.data_ptr(), (size_t)ws.numel(), stream);
  }
  if (rc == OSM_E_LAYOUT) Py_RETURN_NONE;   // tensors that share memory: the Python path says so
  if (rc != OSM_OK) return fail_rc(rc);
  if (scale)
    for (const at::Tensor& t : held) written(t);
  return THPVariable_Wrap(norm);
}

// ---- gated EMA, residual norm, the vocabulary's cross entropy (orthossm_amd/ema.py,
// block_norm.py, linear_loss.py): as above.

osm_seq seq_of(const at::Tensor& t) { return {t.data_ptr(), t.stride(0), t.dim() == 3 ? t.stride(1) : 0}; }

// Rows of contiguous elements that the kernels address, of one float type.
bool ema_tensor(const at::Tensor& t, int64_t dim) {
  if (!t.is_cuda() || !(is_f32(t) || is_bf16(t)) || t.dim() != dim || t.size(dim - 1) < 1 || (t.stride(dim - 1) != 1 && t.size(dim - 1) > 1))
    return false;
  for (int64_t i = 0; i < dim - 1; ++i)
    if (t.stride(i) < 0) return false;
  return true;
}
bool alike(const at::Tensor& t, const at::Tensor& x) {
  return t.scalar_type() == x.scalar_type() && t.sizes() == x.sizes() && t.device() == x.device();
}

bool ema_lengths(const at::Tensor& t, const at::Tensor& x) {
  return t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == x.size(0) && t.is_contiguous() && t.device() == x.device();
}

bool ema_state(const at::Tensor& t, const at::Tensor& x) {
  return t.dim() == 2 && t.size(0) == x.size(0) && t.size(1) == x.size(2) && f32_flat(t, t.numel(), x);
}

void ema_args(const at::Tensor& x, const at::Tensor& gate, osm_ema_args* a) {
  a->abi_version = OSM_ABI_VERSION;
  a->dtype = code(x);
  a->B = x.size(0);
  a->S = x.size(1);
  a->D = x.size(2);
  a->x = seq_of(x);
  a->gate = seq_of(gate);
}

// args: x, gate, lengths, state_init.
bool ema_common(PyObject* const* p, osm_ema_args* a, const at::Tensor** x, const at::Tensor** gate) {
  *x = plain(p[0]);
  *gate = plain(p[1]);
  if (!*x || !*gate || !ema_tensor(**x, 3) || !ema_tensor(**gate, 3) || !alike(**gate, **x)) return false;
  ema_args(**x, **gate, a);
  if (p[2] != Py_None) {
    const at::Tensor* t = plain(p[2]);
    if (!t || !ema_lengths(*t, **x)) return false;
    a->lengths = static_cast<const int32_t*>(t->data_ptr());
  }
  if (p[3] != Py_None) {
    const at::Tensor* t = plain(p[3]);
    if (!t || !ema_state(*t, **x)) return false;
    a->state_init = fptr(*t);
  }
  return true;
}

// The forward into new tensors, those of `fin` and `saved` where wanted.
int ema_forward(osm_ema_args& a, const at::Tensor& x, bool want_state, bool save, void* stream, at::Tensor* out, at::Tensor* fin,
                at::Tensor* saved) {
  *out = empty(x.sizes(), x, x.scalar_type());
  a.out = seq_of(*out);
  if (want_state) {
    *fin = empty({a.B, a.D}, x, at::kFloat);
    a.state_out = fptr(*fin);
  }
  if (save) {
    *saved = scratch(lib.ema_saved(&a), x);
    a.saved = static_cast<float*>(saved->data_ptr());
  }
  const at::Tensor ws = scratch(lib.ema_bytes(&a), x);
  return lib.ema_fwd(&a, ws.data_ptr(), (size_t)ws.numel(), stream);
}

// ema_forward(<common 4>, want_state): None, or (out, state | None).
PyObject* run_ema_forward(PyObject* const* p) {
  osm_ema_args a{};
  const at::Tensor *x, *gate;
  if (!ema_common(p, &a, &x, &gate)) Py_RETURN_NONE;
  const bool want_state = PyObject_IsTrue(p[4]) == 1;
  if (PyErr_Occurred()) return nullptr;
  Ref s_obj;
  void* stream;
  const c10::DeviceGuard guard(x->device());
  if (!stream_of(*x, &s_obj, &stream)) return nullptr;
  at::Tensor out, fin, saved;
  int rc;
  {
    const NoGil nogil;
    rc = ema_forward(a, *x, want_state, false, stream, &out, &fin, &saved);
  }
  if (rc != OSM_OK) return fail_rc(rc);
  return Py_BuildValue("(NN)", THPVariable_Wrap(out), wrap_or_none(fin));
}

struct EmaCall {
  osm_ema_args* a;
  void* stream;
  int rc;
};
struct EmaGrad : torch::autograd::Function<EmaGrad> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& gate,
                                                const std::optional<at::Tensor>& init, const std::optional<at::Tensor>& lengths,
                                                EmaCall* c) {
    ctx->set_materialize_grads(false);   // an unused output's gradient stays undefined
    at::Tensor out, fin, saved;
    c->rc = ema_forward(*c->a, x, true, true, c->stream, &out, &fin, &saved);
    ctx->save_for_backward({x, gate, lengths ? *lengths : at::Tensor(), saved});
    ctx->saved_data["need"] =
        (int64_t)(x.requires_grad() | gate.requires_grad() << 1 | (init && init->requires_grad()) << 2);
    return {out, fin};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto t = ctx->get_saved_variables();
    const int64_t need = ctx->saved_data["need"].toInt();
    at::Tensor gr[3];
    {
      const at::NoGradGuard no_grad;
      const at::Tensor &x = t[0], &saved = t[3];
      TORCH_CHECK(ema_tensor(x, 3) && ema_tensor(t[1], 3) && alike(t[1], x) && (!t[2].defined() || ema_lengths(t[2], x)), kAnotherForm,
                  "gated_ema");
      osm_ema_args a{};
      ema_args(x, t[1], &a);
      TORCH_CHECK(saved.scalar_type() == at::kByte && (size_t)saved.numel() == lib.ema_saved(&a) && saved.is_contiguous() &&
                      saved.device() == x.device(),
                  kAnotherForm, "gated_ema");
      if (t[2].defined()) a.lengths = static_cast<const int32_t*>(t[2].data_ptr());
      a.saved = static_cast<float*>(saved.data_ptr());
      const c10::DeviceGuard guard(x.device());
      at::Tensor go = grads[0].defined() ? grads[0] : at::zeros_like(x);
      if (!ema_tensor(go, 3) || !alike(go, x)) go = go.to(x.options()).contiguous();
      const at::Tensor gs = grads[1].defined() ? grads[1].to(at::kFloat).contiguous() : at::Tensor();
      TORCH_CHECK(ema_tensor(go, 3) && alike(go, x) && (!gs.defined() || ema_state(gs, x)), kAnotherForm, "gated_ema");
      osm_ema_bwd_args b{};
      b.grad_out = seq_of(go);
      if (gs.defined()) b.grad_state = fptr(gs);
      for (int i = 0; i < 2; ++i) gr[i] = empty(x.sizes(), x, x.scalar_type());
      b.grad_x = seq_of(gr[0]);
      b.grad_gate = seq_of(gr[1]);
      if (need & 4) {
        gr[2] = empty({a.B, a.D}, x, at::kFloat);
        b.grad_init = fptr(gr[2]);
      }
      const at::Tensor ws = scratch(lib.ema_bwd_bytes(&a), x);
      throw_rc(lib.ema_bwd(&a, &b, ws.data_ptr(), (size_t)ws.numel(), engine_stream(x)));
    }
    torch::autograd::variable_list res(5);
    for (int i = 0; i < 3; ++i)
      if (need >> i & 1) res[i] = gr[i];
    return once(std::move(res), {grads[0], grads[1], t[0], t[1]});
  }
};

// gated_ema(<common 4>): None, or (out, state) with their gradient's function; without one (out, state).
PyObject* run_gated_ema(PyObject* const* p) {
  osm_ema_args a{};
  const at::Tensor *x, *gate;
  if (!ema_common(p, &a, &x, &gate)) Py_RETURN_NONE;
  const std::optional<at::Tensor> lengths = optional_tensor(p[2]), init = optional_tensor(p[3]);
  if (has_tangent(*x) || has_tangent(*gate) || (init && has_tangent(*init))) Py_RETURN_NONE;
  Ref s_obj;
  void* stream;
  const c10::DeviceGuard guard(x->device());
  if (!stream_of(*x, &s_obj, &stream)) return nullptr;
  const bool grad = x->requires_grad() || gate->requires_grad() || (init && init->requires_grad());
  at::Tensor out, fin, saved;
  int rc;
  {
    const NoGil nogil;
    if (grad && at::GradMode::is_enabled()) {
      EmaCall c{&a, stream, OSM_OK};
      const torch::autograd::variable_list res = EmaGrad::apply(*x, *gate, init, lengths, &c);
      out = res[0];
      fin = res[1];
      rc = c.rc;
    } else {
      rc = ema_forward(a, *x, true, false, stream, &out, &fin, &saved);
    }
  }
  if (rc != OSM_OK) return fail_rc(rc);
  return Py_BuildValue("(NN)", THPVariable_Wrap(out), THPVariable_Wrap(fin));
}

// Whether the bytes from the first element to the last of two matrices meet.
bool extents_meet(const at::Tensor& a, const at::Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return false;
  auto end = [](const at::Tensor& t) {
    const int64_t last = (t.size(0) - 1) * t.stride(0) + (t.size(1) - 1) * t.stride(1);
    return static_cast<const char*>(t.data_ptr()) + (last + 1) * (int64_t)t.element_size();
  };
  return a.data_ptr() < end(b) && b.data_ptr() < end(a);
}

// ema_step(x, gate, state, slots): None, or out.
PyObject* run_ema_step(PyObject* const* p) {
  const at::Tensor *x = plain(p[0]), *gate = plain(p[1]), *state = plain(p[2]);
  if (!x || !gate || !state || !ema_tensor(*x, 2) || !ema_tensor(*gate, 2) || !alike(*gate, *x) || state->dim() != 2 || !is_f32(*state) ||
      state->device() != x->device() || state->size(1) != x->size(1) || (state->stride(1) != 1 && state->size(1) > 1) ||
      state->stride(0) < state->size(1) || state->requires_grad() || extents_meet(*x, *state) || extents_meet(*gate, *state))
    Py_RETURN_NONE;
  osm_ema_step_args a{};
  a.abi_version = OSM_ABI_VERSION;
  a.dtype = code(*x);
  a.B = x->size(0);
  a.D = x->size(1);
  a.x = seq_of(*x);
  a.gate = seq_of(*gate);
  a.state = fptr(*state);
  a.state_stride = state->stride(0);
  a.n_slots = state->size(0);
  if (p[3] == Py_None) {
    if (a.n_slots < a.B) Py_RETURN_NONE;
  } else {
    const at::Tensor* s = plain(p[3]);
    if (!s || s->scalar_type() != at::kLong || s->dim() != 1 || s->size(0) != a.B || !s->is_contiguous() || s->device() != x->device())
      Py_RETURN_NONE;
    a.slots = static_cast<const int64_t*>(s->data_ptr());
  }
  Ref s_obj;
  void* stream;
  const c10::DeviceGuard guard(x->device());
  if (!stream_of(*x, &s_obj, &stream)) return nullptr;
  at::Tensor out;
  int rc;
  {
    const NoGil nogil;
    out = empty({a.B, a.D}, *x, x->scalar_type());
    a.out = seq_of(out);
    rc = lib.ema_step(&a, stream);
  }
  if (rc != OSM_OK) return fail_rc(rc);
  written(*state);
  return THPVariable_Wrap(out);
}

// The residual norm's tensors: x, y, gate (or none), scale, weight, bias (or none).
struct Block {
  const at::Tensor* t[6];
  osm_resnorm_args a{};
};

bool block_tensors(Block* k) {
  const at::Tensor *const xp = k->t[0], *const yp = k->t[1], *const gp = k->t[2];
  if (!norm_rows(xp) || !norm_rows(yp) || yp->sizes() != xp->sizes() || yp->device() != xp->device() || (is_f32(*yp) && !is_f32(*xp)) ||
      (gp && (!norm_rows(gp) || !alike(*gp, *yp))))
    return false;
  osm_resnorm_args& a = k->a;
  a.abi_version = OSM_ABI_VERSION;
  a.stream_dtype = code(*xp);
  a.block_dtype = code(*yp);
  a.D = xp->size(xp->dim() - 1);
  a.rows = xp->numel() / a.D;
  a.x = xp->data_ptr();
  a.y = yp->data_ptr();
  a.gate = gp ? gp->data_ptr() : nullptr;
  a.x_stride = a.y_stride = a.gate_stride = a.D;
  const float** to[3] = {&a.scale, &a.weight, &a.bias};
  for (int i = 0; i < 3; ++i) {
    const at::Tensor* w = k->t[3 + i];
    if (!w) continue;
    if (!f32_vec(w, a.D, *xp)) return false;
    *to[i] = fptr(*w);
  }
  return true;
}

at::DimVector stats_size(const at::Tensor& x) {
  at::DimVector s(x.sizes().begin(), x.sizes().end());
  s.back() = 4;
  return s;
}

int block_forward(Block& k, bool stats, void* stream, at::Tensor* r, at::Tensor* n, at::Tensor* st) {
  const at::Tensor &x = *k.t[0], &y = *k.t[1];
  *r = empty(x.sizes(), x, x.scalar_type());
  *n = empty(x.sizes(), x, y.scalar_type());
  k.a.r = r->data_ptr();
  k.a.n = n->data_ptr();
  k.a.r_stride = k.a.n_stride = k.a.D;
  if (stats) {
    *st = empty(stats_size(x), x, at::kFloat);
    k.a.stats = fptr(*st);
  }
  return lib.block_fwd(&k.a, stream);
}

struct BlockCall {
  Block* k;
  void* stream;
  int rc;
};
struct BlockGrad : torch::autograd::Function<BlockGrad> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& y,
                                                const std::optional<at::Tensor>& gate, const std::optional<at::Tensor>& scale,
                                                const std::optional<at::Tensor>& weight, const std::optional<at::Tensor>& bias,
                                                BlockCall* c) {
    ctx->set_materialize_grads(false);   // an unused output's gradient stays undefined
    at::Tensor r, n, st;
    c->rc = block_forward(*c->k, true, c->stream, &r, &n, &st);
    const at::Tensor none;
    ctx->save_for_backward({x, y, gate ? *gate : none, scale ? *scale : none, weight ? *weight : none, st});
    int64_t need = x.requires_grad() | y.requires_grad() << 1;
    const std::optional<at::Tensor>* rest[4] = {&gate, &scale, &weight, &bias};
    for (int i = 0; i < 4; ++i) need |= (int64_t)(*rest[i] && (*rest[i])->requires_grad()) << (2 + i);
    ctx->saved_data["need"] = need;
    ctx->saved_data["flags"] = (int64_t)c->k->a.flags;
    return {r, n};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto t = ctx->get_saved_variables();
    const int64_t need = ctx->saved_data["need"].toInt();
    torch::autograd::variable_list res(7);
    {
      const at::NoGradGuard no_grad;
      Block k;
      for (int i = 0; i < 5; ++i) k.t[i] = t[i].defined() ? &t[i] : nullptr;
      k.t[5] = nullptr;
      const bool inputs = block_tensors(&k);
      TORCH_CHECK(inputs && f32_flat(t[5], 4 * k.a.rows, t[0]), kAnotherForm, "residual_norm");
      const at::Tensor &x = t[0], &y = t[1];
      k.a.flags = (int32_t)ctx->saved_data["flags"].toInt();
      k.a.stats = fptr(t[5]);
      const c10::DeviceGuard guard(x.device());
      osm_resnorm_bwd_args b{};
      at::Tensor g[2];
      const void** const at_g[2] = {&b.grad_r, &b.grad_n};
      for (int i = 0; i < 2; ++i) {
        if (!grads[i].defined()) continue;
        const at::Tensor& like = i ? y : x;
        g[i] = norm_grad_form(grads[i], like) ? grads[i] : grads[i].to(like.options()).contiguous();
        TORCH_CHECK(norm_grad_form(g[i], like), kAnotherForm, "residual_norm");
        *at_g[i] = g[i].data_ptr();
      }
      b.grad_r_stride = b.grad_n_stride = b.grad_x_stride = b.grad_y_stride = b.grad_gate_stride = k.a.D;
      void** const rows[3] = {&b.grad_x, &b.grad_y, &b.grad_gate};
      float** const sums[3] = {&b.grad_scale, &b.grad_weight, &b.grad_bias};
      for (int i = 0; i < 3; ++i) {
        if (need >> i & 1) {
          res[i] = empty(x.sizes(), x, t[i].scalar_type());
          *rows[i] = res[i].data_ptr();
        }
        if (need >> (3 + i) & 1) {
          res[3 + i] = empty({k.a.D}, x, at::kFloat);
          *sums[i] = fptr(res[3 + i]);
        }
      }
      const at::Tensor ws = scratch(lib.block_bwd_bytes(&k.a), x);
      throw_rc(lib.block_bwd(&k.a, &b, ws.data_ptr(), (size_t)ws.numel(), engine_stream(x)));
    }
    return once(std::move(res), {grads[0], grads[1], t[0], t[1], t[2], t[3], t[4]});
  }
};

// residual_norm(x, y, gate, scale, weight, bias, flags, eps): None, or (r, n) with their gradient's function.
PyObject* run_residual_norm(PyObject* const* p) {
  Block k;
  for (int i = 0; i < 6; ++i) {
    k.t[i] = p[i] == Py_None ? nullptr : plain(p[i]);
    if (!k.t[i] && (i < 2 || p[i] != Py_None)) Py_RETURN_NONE;
  }
  if (!block_tensors(&k) || !as_float(p[7], &k.a.eps)) Py_RETURN_NONE;
  k.a.flags = (int32_t)PyLong_AsLong(p[6]);
  if (PyErr_Occurred()) return nullptr;
  bool grad = false;
  for (const at::Tensor* t : k.t) {
    if (t && has_tangent(*t)) Py_RETURN_NONE;
    grad = grad || (t && t->requires_grad());
  }
  const at::Tensor &x = *k.t[0], &y = *k.t[1];
  Ref s_obj;
  void* stream;
  const c10::DeviceGuard guard(x.device());
  if (!stream_of(x, &s_obj, &stream)) return nullptr;
  at::Tensor r, n, st;
  int rc;
  {
    const NoGil nogil;
    if (grad && at::GradMode::is_enabled()) {
      BlockCall c{&k, stream, OSM_OK};
      const torch::autograd::variable_list res =
          BlockGrad::apply(x, y, optional_tensor(p[2]), optional_tensor(p[3]), optional_tensor(p[4]), optional_tensor(p[5]), &c);
      r = res[0];
      n = res[1];
      rc = c.rc;
    } else {
      rc = block_forward(k, false, stream, &r, &n, &st);
    }
  }
  if (rc != OSM_OK) return fail_rc(rc);
  return Py_BuildValue("(NN)", THPVariable_Wrap(r), THPVariable_Wrap(n));
}

// The cross entropy's tensors: hidden [.., D], weight [V,D], targets.
bool loss_tensors(const at::Tensor& h, const at::Tensor& w, const at::Tensor& t, osm_loss_args* a) {
  if (!norm_rows(&h) || !w.is_cuda() || w.dim() != 2 || w.scalar_type() != h.scalar_type() || w.device() != h.device() ||
      w.size(0) < 1 || w.size(1) != h.size(h.dim() - 1) || !w.is_contiguous() || t.scalar_type() != at::kLong || t.device() != h.device() ||
      !t.is_contiguous() || t.sizes() != h.sizes().slice(0, h.dim() - 1))
    return false;
  a->abi_version = OSM_ABI_VERSION;
  a->dtype = code(h);
  a->D = w.size(1);
  a->V = w.size(0);
  a->N = t.numel();
  a->hidden = h.data_ptr();
  a->weight = w.data_ptr();
  a->hidden_stride = a->weight_stride = a->D;
  a->targets = static_cast<const int64_t*>(t.data_ptr());
  return true;
}

// 0: every token's loss, 1: their sum, 2: their mean
int loss_forward(osm_loss_args& a, const at::Tensor& h, const at::Tensor& t, int64_t how, void* stream, at::Tensor* loss, at::Tensor* lse,
                 at::Tensor* count) {
  at::Tensor losses = empty(t.sizes(), h, at::kFloat);
  *lse = empty(t.sizes(), h, at::kFloat);
  a.losses = fptr(losses);
  a.lse = fptr(*lse);
  if (how == 0) {
    *loss = losses;
  } else {
    *loss = empty({}, h, at::kFloat);
    a.loss = fptr(*loss);
  }
  if (how == 2) {
    a.flags = OSM_LOSS_MEAN;
    *count = empty({}, h, at::kFloat);
    a.count = fptr(*count);
  }
  const at::Tensor ws = scratch(lib.loss_bytes(&a), h);
  return lib.loss_fwd(&a, ws.data_ptr(), (size_t)ws.numel(), stream);
}

struct LossCall {
  osm_loss_args* a;
  int64_t how;
  void* stream;
  int rc;
};
struct LossGrad : torch::autograd::Function<LossGrad> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& h, const at::Tensor& w, const at::Tensor& t,
                            LossCall* c) {
    at::Tensor loss, lse, count;
    c->rc = loss_forward(*c->a, h, t, c->how, c->stream, &loss, &lse, &count);
    ctx->save_for_backward({h, w, t, lse, count});
    ctx->saved_data["need"] = (int64_t)(h.requires_grad() | w.requires_grad() << 1);
    ctx->saved_data["each"] = c->how == 0;
    ctx->saved_data["ignore"] = c->a->ignore_index;
    return loss;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto t = ctx->get_saved_variables();
    const int64_t need = ctx->saved_data["need"].toInt();
    const bool each = ctx->saved_data["each"].toBool();
    torch::autograd::variable_list res(4);
    {
      const at::NoGradGuard no_grad;
      const at::Tensor &h = t[0], &w = t[1], &lse = t[3];
      osm_loss_args a{};
      TORCH_CHECK(loss_tensors(h, w, t[2], &a) && f32_flat(lse, a.N, h) && (!t[4].defined() || f32_flat(t[4], 1, h)), kAnotherForm,
                  "linear_cross_entropy");
      a.ignore_index = ctx->saved_data["ignore"].toInt();
      a.lse = fptr(lse);
      const c10::DeviceGuard guard(h.device());
      const at::Tensor g = grads[0].to(at::kFloat).contiguous();
      TORCH_CHECK(f32_flat(g, each ? a.N : 1, h), kAnotherForm, "linear_cross_entropy");
      osm_loss_bwd_args b{};
      (each ? b.grad_losses : b.grad) = fptr(g);
      if (t[4].defined()) b.count = fptr(t[4]);
      void** const to[2] = {&b.grad_hidden, &b.grad_weight};
      for (int i = 0; i < 2; ++i)
        if (need >> i & 1) {
          res[i] = empty(t[i].sizes(), h, h.scalar_type());
          *to[i] = res[i].data_ptr();
        }
      const at::Tensor ws = scratch(lib.loss_bwd_bytes(&a), h);
      throw_rc(lib.loss_bwd(&a, &b, ws.data_ptr(), (size_t)ws.numel(), engine_stream(h)));
    }
    return once(std::move(res), {grads[0], t[0], t[1]});
  }
};

// linear_cross_entropy(hidden, weight, targets, ignore_index, how): None, or the loss with its gradient's function.
PyObject* run_linear_loss(PyObject* const* p) {
  const at::Tensor *h = plain(p[0]), *w = plain(p[1]), *t = plain(p[2]);
  osm_loss_args a{};
  int64_t how;
  if (!h || !w || !t || !loss_tensors(*h, *w, *t, &a) || !as_int(p[3], &a.ignore_index) || !as_int(p[4], &how)) Py_RETURN_NONE;
  if (has_tangent(*h) || has_tangent(*w)) Py_RETURN_NONE;
  Ref s_obj;
  void* stream;
  const c10::DeviceGuard guard(h->device());
  if (!stream_of(*h, &s_obj, &stream)) return nullptr;
  at::Tensor loss, lse, count;
  int rc;
  {
    const NoGil nogil;
    if ((h->requires_grad() || w->requires_grad()) && at::GradMode::is_enabled()) {
      LossCall c{&a, how, stream, OSM_OK};
      loss = LossGrad::apply(*h, *w, *t, &c);
      rc = c.rc;
    } else {
      rc = loss_forward(a, *h, *t, how, stream, &loss, &lse, &count);
    }
  }
  if (rc != OSM_OK) return fail_rc(rc);
  return THPVariable_Wrap(loss);
}

// Runs a function under the argument count and the C++ exceptions of ATen.
template <int N, typename F>
PyObject* guarded(PyObject* const* args, Py_ssize_t n, F f) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "takes %d arguments, got %zd", N, n);
    return nullptr;
  }
  if (!check) {
    PyErr_SetString(PyExc_RuntimeError, "init() has not been called");
    return nullptr;
  }
  HANDLE_TH_ERRORS   // C++ exceptions become torch's own Python ones
  return f(args);
  END_HANDLE_TH_ERRORS
}

PyObject* py_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded<14>(a, n, [](PyObject* const* p) { return run_forward(p, false); });
}
PyObject* py_ttt(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded<15>(a, n, [](PyObject* const* p) { return run_forward(p, true); });
}
PyObject* py_backward(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded<14>(a, n, run_backward); }
PyObject* py_v10(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded<18>(a, n, run_v10); }
PyObject* py_v10_backward(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded<7>(a, n, run_v10_backward); }
PyObject* py_lut(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded<10>(a, n, run_lut); }
PyObject* py_engine(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded<9>(a, n, run_engine); }

PyObject* py_delta_forward(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded<10>(a, n, run_delta_forward); }
PyObject* py_delta_backward(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded<11>(a, n, run_delta_backward); }
PyObject* py_gated_delta(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded<9>(a, n, run_gated_delta); }
PyObject* py_delta_step(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded<8>(a, n, run_delta_step); }
PyObject* py_norm_forward(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded<5>(a, n, run_norm_forward); }
PyObject* py_norm_backward(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded<8>(a, n, run_norm_backward); }
PyObject* py_layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded<4>(a, n, run_layer_norm); }
PyObject* py_clip(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded<4>(a, n, run_clip); }
PyObject* py_ema_forward(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded<5>(a, n, run_ema_forward); }
PyObject* py_gated_ema(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded<4>(a, n, run_gated_ema); }
PyObject* py_ema_step(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded<4>(a, n, run_ema_step); }
PyObject* py_residual_norm(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded<8>(a, n, run_residual_norm); }
PyObject* py_linear_loss(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded<5>(a, n, run_linear_loss); }

// init(addresses of the library's functions in the order of Lib, raw_stream, ws_cache, workspace, check)
PyObject* py_init(PyObject*, PyObject* args) {
  PyObject *addr, *rs, *wc, *wf, *ck;
  if (!PyArg_ParseTuple(args, "O!OO!OO", &PyTuple_Type, &addr, &rs, &PyDict_Type, &wc, &wf, &ck)) return nullptr;
  void* f[kFunctions];
  if (PyTuple_GET_SIZE(addr) != kFunctions) {
    PyErr_Format(PyExc_ValueError, "%d addresses are expected", kFunctions);
    return nullptr;
  }
  for (int i = 0; i < kFunctions; ++i) f[i] = PyLong_AsVoidPtr(PyTuple_GET_ITEM(addr, i));
  if (PyErr_Occurred()) return nullptr;
  lib.workspace_bytes = reinterpret_cast<decltype(lib.workspace_bytes)>(f[0]);
  lib.fwd = reinterpret_cast<decltype(lib.fwd)>(f[1]);
  lib.ttt = reinterpret_cast<decltype(lib.ttt)>(f[2]);
  lib.bwd = reinterpret_cast<decltype(lib.bwd)>(f[3]);
  lib.v10 = reinterpret_cast<decltype(lib.v10)>(f[4]);
  lib.v10_bwd = reinterpret_cast<decltype(lib.v10_bwd)>(f[5]);
  lib.lut_bytes = reinterpret_cast<decltype(lib.lut_bytes)>(f[6]);
  lib.lut_ws = reinterpret_cast<decltype(lib.lut_ws)>(f[7]);
  lib.engine_bytes = reinterpret_cast<decltype(lib.engine_bytes)>(f[8]);
  lib.engine = reinterpret_cast<decltype(lib.engine)>(f[9]);
  lib.stream_is_capturing = reinterpret_cast<decltype(lib.stream_is_capturing)>(f[10]);
  lib.delta_saved = reinterpret_cast<decltype(lib.delta_saved)>(f[11]);
  lib.delta_bytes = reinterpret_cast<decltype(lib.delta_bytes)>(f[12]);
  lib.delta_fwd = reinterpret_cast<decltype(lib.delta_fwd)>(f[13]);
  lib.delta_bwd_bytes = reinterpret_cast<decltype(lib.delta_bwd_bytes)>(f[14]);
  lib.delta_bwd = reinterpret_cast<decltype(lib.delta_bwd)>(f[15]);
  lib.delta_step = reinterpret_cast<decltype(lib.delta_step)>(f[16]);
  lib.norm_fwd = reinterpret_cast<decltype(lib.norm_fwd)>(f[17]);
  lib.norm_bwd_bytes = reinterpret_cast<decltype(lib.norm_bwd_bytes)>(f[18]);
  lib.norm_bwd = reinterpret_cast<decltype(lib.norm_bwd)>(f[19]);
  lib.clip_bytes = reinterpret_cast<decltype(lib.clip_bytes)>(f[20]);
  lib.clip = reinterpret_cast<decltype(lib.clip)>(f[21]);
  lib.ema_saved = reinterpret_cast<decltype(lib.ema_saved)>(f[22]);
  lib.ema_bytes = reinterpret_cast<decltype(lib.ema_bytes)>(f[23]);
  lib.ema_fwd = reinterpret_cast<decltype(lib.ema_fwd)>(f[24]);
  lib.ema_bwd_bytes = reinterpret_cast<decltype(lib.ema_bwd_bytes)>(f[25]);
  lib.ema_bwd = reinterpret_cast<decltype(lib.ema_bwd)>(f[26]);
  lib.ema_step = reinterpret_cast<decltype(lib.ema_step)>(f[27]);
  lib.block_fwd = reinterpret_cast<decltype(lib.block_fwd)>(f[28]);
  lib.block_bwd_bytes = reinterpret_cast<decltype(lib.block_bwd_bytes)>(f[29]);
  lib.block_bwd = reinterpret_cast<decltype(lib.block_bwd)>(f[30]);
  lib.loss_bytes = reinterpret_cast<decltype(lib.loss_bytes)>(f[31]);
  lib.loss_fwd = reinterpret_cast<decltype(lib.loss_fwd)>(f[32]);
  lib.loss_bwd_bytes = reinterpret_cast<decltype(lib.loss_bwd_bytes)>(f[33]);
  lib.loss_bwd = reinterpret_cast<decltype(lib.loss_bwd)>(f[34]);
  PyObject** slots[4] = {&raw_stream, &ws_cache, &workspace, &check};
  PyObject* vals[4] = {rs, wc, wf, ck};
  for (int i = 0; i < 4; ++i) {
    Py_INCREF(vals[i]);
    PyObject* old = *slots[i];
    *slots[i] = vals[i];
    Py_XDECREF(old);
  }
  Py_RETURN_NONE;
}

template <typename F>
PyCFunction fast(F f) {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}

PyMethodDef methods[] = {
    {"init", py_init, METH_VARARGS, nullptr},
    {"forward", fast(py_forward), METH_FASTCALL, nullptr},
    {"ttt", fast(py_ttt), METH_FASTCALL, nullptr},
    {"backward", fast(py_backward), METH_FASTCALL, nullptr},
    {"v10", fast(py_v10), METH_FASTCALL, nullptr},
    {"v10_backward", fast(py_v10_backward), METH_FASTCALL, nullptr},
    {"lut_forward", fast(py_lut), METH_FASTCALL, nullptr},
    {"engine", fast(py_engine), METH_FASTCALL, nullptr},
    {"delta_forward", fast(py_delta_forward), METH_FASTCALL, nullptr},
    {"delta_backward", fast(py_delta_backward), METH_FASTCALL, nullptr},
    {"gated_delta", fast(py_gated_delta), METH_FASTCALL, nullptr},
    {"delta_step", fast(py_delta_step), METH_FASTCALL, nullptr},
    {"norm_forward", fast(py_norm_forward), METH_FASTCALL, nullptr},
    {"norm_backward", fast(py_norm_backward), METH_FASTCALL, nullptr},
    {"layer_norm", fast(py_layer_norm), METH_FASTCALL, nullptr},
    {"clip", fast(py_clip), METH_FASTCALL, nullptr},
    {"ema_forward", fast(py_ema_forward), METH_FASTCALL, nullptr},
    {"gated_ema", fast(py_gated_ema), METH_FASTCALL, nullptr},
    {"ema_step", fast(py_ema_step), METH_FASTCALL, nullptr},
    {"residual_norm", fast(py_residual_norm), METH_FASTCALL, nullptr},
    {"linear_loss", fast(py_linear_loss), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "osm_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// built_for: the torch version and the Python minor version of the build.
PyMODINIT_FUNC PyInit_osm_torch(void) {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddObject(m, "built_for", Py_BuildValue("(si)", TORCH_VERSION, PY_VERSION_HEX >> 16)) != 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
