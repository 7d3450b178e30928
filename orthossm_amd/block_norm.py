"""A block's residual update between its two norms over the C ABI (HIP kernels
on gfx950).

    r = x + scale * sigmoid(gate) * N(y),   n = N(r) * weight + bias     over the last axis

x is the residual stream and y what a block made of it: N(y) is the norm after
the block (``norm_y`` false: y itself), scale and sigmoid(gate) weigh what is
added, n is what the next block reads.  N is the layer norm without parameters
or, with ``rms``, v / sqrt(mean(v^2) + eps).

``residual_norm``           the differentiable op: (r, n), gradients to x, y,
                            gate, scale, weight and bias.
``residual_norm_forward``   (r, n, stats).
``residual_norm_backward``  the six gradients from dL/dr and dL/dn.

x [..., D] and y, gate of the same shape, fp32 or bf16 (other types go to fp32)
with contiguous rows (others are copied first); y and gate of one type (mixed:
fp32), x of the same or fp32 (bf16 x with fp32 y: goes to fp32).  r has x's type,
n has y's.  scale, weight, bias [D] or None; statistics, parameters and their
gradients are fp32.  All run on the current torch stream of x's device and never
synchronise the host.  There is no CPU path.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _native as nat
from .delta import _scratch, differentiable, on_device
from .norm import _matrix, _param
from .ops import _current_stream, _dtype_code, _fast

_TYPES = (torch.float32, torch.bfloat16)


def _flags(norm_y, rms) -> int:
    return (nat.RESNORM_NORM_Y if norm_y else 0) | (nat.RESNORM_RMS if rms else 0)


def _prepare(x, y, gate, scale, weight, bias, norm_y, rms, eps):
    if not isinstance(x, torch.Tensor) or x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x must be a [..., D] tensor with D >= 1")
    if x.device.type != "cuda":
        raise RuntimeError(f"orthossm_amd runs on a ROCm GPU only; x is on {x.device}")
    for name, t in (("y", y), ("gate", gate)):
        if t is None and name == "gate":
            continue
        if not isinstance(t, torch.Tensor) or t.shape != x.shape or t.device != x.device:
            raise ValueError(f"{name} must be a tensor of shape {tuple(x.shape)} on {x.device}")
    if y.dtype not in _TYPES or (gate is not None and gate.dtype != y.dtype):
        y, gate = y.float(), None if gate is None else gate.float()
    if x.dtype not in _TYPES or y.dtype == torch.float32:
        x = x.float()
    D = x.shape[-1]
    scale, weight, bias = (_param(t, D, x.device, name) for name, t in (("scale", scale), ("weight", weight), ("bias", bias)))
    mx, my, mg = _matrix(x), _matrix(y), None if gate is None else _matrix(gate)
    a = nat.ResnormArgs()
    a.abi_version = nat.ABI_VERSION
    a.flags = _flags(norm_y, rms)
    a.stream_dtype, a.block_dtype = _dtype_code(x.dtype), _dtype_code(y.dtype)
    a.rows, a.D, a.eps = mx.shape[0], D, float(eps)
    a.x, a.x_stride = mx.data_ptr(), mx.stride(0)
    a.y, a.y_stride = my.data_ptr(), my.stride(0)
    if mg is not None:
        a.gate, a.gate_stride = mg.data_ptr(), mg.stride(0)
    for name, t in (("scale", scale), ("weight", weight), ("bias", bias)):
        setattr(a, name, None if t is None else t.data_ptr())
    return a, (x, y, gate, scale, weight, bias), (mx, my, mg)


def _forward(x, y, gate, scale, weight, bias, norm_y, rms, eps, stats: bool):
    lib = nat.load()
    a, ins, keep = _prepare(x, y, gate, scale, weight, bias, norm_y, rms, eps)
    x, y = ins[:2]
    dev = x.device
    r, n = torch.empty(x.shape, dtype=x.dtype, device=dev), torch.empty(x.shape, dtype=y.dtype, device=dev)
    a.r, a.r_stride, a.n, a.n_stride = r.data_ptr(), a.D, n.data_ptr(), a.D
    st = torch.empty((*x.shape[:-1], 4), dtype=torch.float32, device=dev) if stats else None
    a.stats = st.data_ptr() if stats else None
    with on_device(dev):
        nat.check(lib.osm_residual_norm_fwd(ctypes.byref(a), ctypes.c_void_p(_current_stream(dev))))
    del keep
    return r, n, st, ins


def residual_norm_forward(x: torch.Tensor, y: torch.Tensor, weight: torch.Tensor | None = None,
                          bias: torch.Tensor | None = None, *, gate: torch.Tensor | None = None,
                          scale: torch.Tensor | None = None, norm_y: bool = True, rms: bool = False, eps: float = 1e-5):
    """(r in x's type, n in y's, stats fp32 of x's shape with 4 in place of D:
    mean and 1 / spread of y, then of r)."""
    return _forward(x, y, gate, scale, weight, bias, norm_y, rms, eps, True)[:3]


def residual_norm_backward(grad_r: torch.Tensor | None, grad_n: torch.Tensor | None, x: torch.Tensor, y: torch.Tensor,
                           stats: torch.Tensor, weight: torch.Tensor | None = None, *, gate: torch.Tensor | None = None,
                           scale: torch.Tensor | None = None, norm_y: bool = True, rms: bool = False,
                           need=(True,) * 6):
    """(grad_x in x's type, grad_y and grad_gate in y's, grad_scale, grad_weight,
    grad_bias fp32) from dL/dr and dL/dn (None: zeros), the forward's inputs and
    what it gave; None for what ``need`` (in that order) leaves out and for the
    gate's where there is none."""
    lib = nat.load()
    a, (x, y, gate, *_), keep = _prepare(x, y, gate, scale, weight, None, norm_y, rms, 0.0)
    dev, D = x.device, a.D
    if not isinstance(stats, torch.Tensor) or stats.shape != (*x.shape[:-1], 4) or stats.dtype != torch.float32 or \
            stats.device != dev:
        raise ValueError(f"stats must be a float32 tensor of shape {(*x.shape[:-1], 4)} on {dev}")
    stats = stats.contiguous()
    a.stats = stats.data_ptr()
    b = nat.ResnormBwdArgs()
    held = []
    for name, t, like in (("grad_r", grad_r, x), ("grad_n", grad_n, y)):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor) or t.shape != x.shape:
            raise ValueError(f"{name} must be a tensor of shape {tuple(x.shape)}")
        held.append(_matrix(t.to(device=dev, dtype=like.dtype)))
        setattr(b, name, held[-1].data_ptr())
        setattr(b, name + "_stride", held[-1].stride(0))
    grads = []
    for name, like, n in zip(("grad_x", "grad_y", "grad_gate"), (x, y, gate), need):
        t = torch.empty(x.shape, dtype=like.dtype, device=dev) if n and like is not None else None
        if t is not None:
            setattr(b, name, t.data_ptr())
            setattr(b, name + "_stride", D)
        grads.append(t)
    for name, n in zip(("grad_scale", "grad_weight", "grad_bias"), need[3:]):
        grads.append(torch.empty(D, dtype=torch.float32, device=dev) if n else None)
        setattr(b, name, grads[-1].data_ptr() if n else None)
    ws = _scratch(lib.osm_residual_norm_bwd_workspace_bytes(ctypes.byref(a)), dev)
    with on_device(dev):
        nat.check(lib.osm_residual_norm_bwd(ctypes.byref(a), ctypes.byref(b), ctypes.c_void_p(ws.data_ptr()), ws.numel(),
                                            ctypes.c_void_p(_current_stream(dev))))
    del keep
    return tuple(grads)


class _ResidualNormFunction(torch.autograd.Function):
    """Saves the inputs and the statistics."""

    @staticmethod
    def forward(ctx, x, y, gate, scale, weight, bias, norm_y, rms, eps):
        ctx.set_materialize_grads(False)   # an unused output's gradient stays None
        r, n, stats, ins = _forward(x, y, gate, scale, weight, bias, norm_y, rms, eps, True)
        ctx.save_for_backward(*ins[:5], stats)
        ctx.form = dict(norm_y=norm_y, rms=rms)
        ctx.types = [None if t is None else t.dtype for t in (x, y, gate, scale, weight, bias)]
        return r, n

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_r, grad_n):
        x, y, gate, scale, weight, stats = ctx.saved_tensors
        grads = residual_norm_backward(grad_r, grad_n, x, y, stats, weight, gate=gate, scale=scale,
                                       need=ctx.needs_input_grad[:6], **ctx.form)
        return (*(None if t is None else t.to(dt) for t, dt in zip(grads, ctx.types)), None, None, None)


def residual_norm(x: torch.Tensor, y: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                  *, gate: torch.Tensor | None = None, scale: torch.Tensor | None = None, norm_y: bool = True,
                  rms: bool = False, eps: float = 1e-5):
    """(r, n): the residual stream after a block's output y, and its norm,
    differentiable in x, y, gate, scale, weight and bias."""
    fast = _fast()
    if fast is not None:
        res = fast.residual_norm(x, y, gate, scale, weight, bias, _flags(norm_y, rms), eps)
        if res is not None:
            return res
    if differentiable(x, y, gate, scale, weight, bias):
        return _ResidualNormFunction.apply(x, y, gate, scale, weight, bias, bool(norm_y), bool(rms), eps)
    return _forward(x, y, gate, scale, weight, bias, norm_y, rms, eps, False)[:2]
