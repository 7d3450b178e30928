"""Layer norm over the C ABI (HIP kernels on gfx950).

    y = (x - mean) / sqrt(variance + eps) * weight + bias     over the last axis

``layer_norm``           the differentiable op: gradients to x, weight and bias.
``layer_norm_forward``   (y, mean, rstd).
``layer_norm_backward``  (grad_x, grad_weight, grad_bias) from dL/dy.

x [..., D] fp32 or bf16 (other types go to fp32) with contiguous rows (others
are copied first), weight and bias [D] or None; statistics, parameters and
their gradients are fp32.  All run on the current torch stream of x's device
and never synchronise the host.  There is no CPU path.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _native as nat
from .delta import _dest, _scratch, apart, differentiable, on_device, written
from .ops import _current_stream, _dtype_code, _fast


def _matrix(t: torch.Tensor) -> torch.Tensor:
    """[rows, D] with contiguous elements and one row stride, a view where t's layout allows it."""
    if t.dim() == 1:
        t = t.unsqueeze(0)
    if t.stride(-1) != 1 and t.shape[-1] != 1:
        t = t.contiguous()
    try:
        return t.view(-1, t.shape[-1])
    except RuntimeError:
        return t.contiguous().view(-1, t.shape[-1])


def _param(t, D: int, dev, name: str) -> torch.Tensor | None:
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or tuple(t.shape) != (D,):
        raise ValueError(f"{name} must be a tensor of shape ({D},)")
    return t.to(device=dev, dtype=torch.float32).contiguous()


def _prepare(x, weight, bias, eps):
    if not isinstance(x, torch.Tensor) or x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x must be a [..., D] tensor with D >= 1")
    if x.device.type != "cuda":
        raise RuntimeError(f"orthossm_amd runs on a ROCm GPU only; x is on {x.device}")
    if x.dtype not in (torch.float32, torch.bfloat16):
        x = x.float()
    D = x.shape[-1]
    weight, bias = _param(weight, D, x.device, "weight"), _param(bias, D, x.device, "bias")
    rows = _matrix(x)
    a = nat.NormArgs()
    a.abi_version, a.dtype = nat.ABI_VERSION, _dtype_code(x.dtype)
    a.rows, a.D, a.eps = rows.shape[0], D, float(eps)
    a.x, a.x_stride = rows.data_ptr(), rows.stride(0)
    a.weight = weight.data_ptr() if weight is not None else None
    a.bias = bias.data_ptr() if bias is not None else None
    return a, x, (rows, weight, bias)


def _forward(x, weight, bias, eps, out, stats: bool):
    fast = _fast()
    if fast is not None and out is None:
        res = fast.norm_forward(x, weight, bias, eps, stats)
        if res is not None:
            return res
    lib = nat.load()
    a, x, keep = _prepare(x, weight, bias, eps)
    dev, given = x.device, out
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=dev)
    else:
        _dest(out, x.shape, x.dtype, dev, "out")
        rows, weight, bias = keep
        apart("out", out.view(rows.shape), dict(x=rows, weight=weight, bias=bias), "x")
    a.y, a.y_stride = out.data_ptr(), a.D
    mean = rstd = None
    if stats:
        mean, rstd = (torch.empty(x.shape[:-1], dtype=torch.float32, device=dev) for _ in range(2))
        a.mean, a.rstd = mean.data_ptr(), rstd.data_ptr()
    with on_device(dev):
        nat.check(lib.osm_layer_norm_fwd(ctypes.byref(a), ctypes.c_void_p(_current_stream(dev))))
    written(given)
    del keep
    return out, mean, rstd


def layer_norm_forward(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, *,
                       eps: float = 1e-5, out: torch.Tensor | None = None):
    """(y in x's type, mean and rstd fp32 of x's shape without the last axis).
    ``out`` (contiguous; may be x, else in no argument's memory) receives y
    instead of a new tensor."""
    return _forward(x, weight, bias, eps, out, True)


def layer_norm_backward(grad_y: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                        weight: torch.Tensor | None = None, *, need_x: bool = True, need_weight: bool = True,
                        need_bias: bool = True):
    """(grad_x in x's type, grad_weight, grad_bias fp32), None for what is not
    needed, from dL/dy, x and what the forward gave."""
    fast = _fast()
    if fast is not None:
        res = fast.norm_backward(grad_y, x, mean, rstd, weight, need_x, need_weight, need_bias)
        if res is not None:
            return res
    lib = nat.load()
    a, x, keep = _prepare(x, weight, None, 0.0)
    dev, D = x.device, a.D
    if not isinstance(grad_y, torch.Tensor) or grad_y.shape != x.shape:
        raise ValueError(f"grad_y must be a tensor of shape {tuple(x.shape)}")
    stats = []
    for name, t in (("mean", mean), ("rstd", rstd)):
        if not isinstance(t, torch.Tensor) or t.shape != x.shape[:-1] or t.dtype != torch.float32 or t.device != dev:
            raise ValueError(f"{name} must be a float32 tensor of shape {tuple(x.shape[:-1])} on {dev}")
        stats.append(t.contiguous())
    a.mean, a.rstd = (t.data_ptr() for t in stats)
    go = _matrix(grad_y.to(device=dev, dtype=x.dtype))
    gx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_x else None
    gw = torch.empty(D, dtype=torch.float32, device=dev) if need_weight else None
    gb = torch.empty(D, dtype=torch.float32, device=dev) if need_bias else None
    b = nat.NormBwdArgs()
    b.grad_y, b.grad_y_stride = go.data_ptr(), go.stride(0)
    if need_x:
        b.grad_x, b.grad_x_stride = gx.data_ptr(), D
    b.grad_weight = gw.data_ptr() if need_weight else None
    b.grad_bias = gb.data_ptr() if need_bias else None
    ws = _scratch(lib.osm_layer_norm_bwd_workspace_bytes(ctypes.byref(a)), dev)
    with on_device(dev):
        nat.check(lib.osm_layer_norm_bwd(ctypes.byref(a), ctypes.byref(b), ctypes.c_void_p(ws.data_ptr()), ws.numel(),
                                         ctypes.c_void_p(_current_stream(dev))))
    del keep
    return gx, gw, gb


class _LayerNormFunction(torch.autograd.Function):
    """Saves x, the statistics and the weight."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = _forward(x, weight, bias, eps, None, True)
        ctx.save_for_backward(x, mean, rstd, weight)
        ctx.types = [None if t is None else t.dtype for t in (x, weight, bias)]
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y):
        x, mean, rstd, weight = ctx.saved_tensors
        need = ctx.needs_input_grad
        grads = layer_norm_backward(grad_y, x, mean, rstd, weight, need_x=need[0], need_weight=need[1],
                                    need_bias=need[2])
        return (*(None if t is None else t.to(dt) for t, dt in zip(grads, ctx.types)), None)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, *,
               eps: float = 1e-5) -> torch.Tensor:
    """Layer norm over the last axis, differentiable in x, weight and bias."""
    fast = _fast()
    if fast is not None:
        y = fast.layer_norm(x, weight, bias, eps)
        if y is not None:
            return y
    if differentiable(x, weight, bias):
        return _LayerNormFunction.apply(x, weight, bias, eps)
    return _forward(x, weight, bias, eps, None, False)[0]
