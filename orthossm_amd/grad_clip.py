"""The global gradient norm over the C ABI (HIP kernels on gfx950).

``grad_norm``       sqrt of the sum of squares over all elements of many tensors.
``clip_grad_norm``  the same, and every tensor times min(1, max_norm / (norm + eps)) in place.

Tensors are fp32 or bf16 in any mix, of any sizes, on one device; those that are
clipped share no memory.  Sums are held in double; the norm stays on the device,
so nothing synchronises the host.  A NaN norm makes every element NaN, an
infinite one makes finite elements 0 and infinite ones NaN.  There is no CPU path.
"""
from __future__ import annotations

import ctypes
from typing import Iterable

import torch

from . import _native as nat
from .delta import _scratch, on_device, written
from .ops import _current_stream, _dtype_code, _fast


def _dense(t: torch.Tensor) -> bool:
    """Whether t's elements are numel() consecutive ones of memory, in any order of its axes."""
    n = 1
    for stride, size in sorted((s, z) for s, z in zip(t.stride(), t.shape) if z != 1):
        if stride != n:
            return False
        n *= size
    return True


def _share_memory(tensors) -> bool:
    """Whether an element of these tensors (none of them empty) is in two places:
    for dense ones by their extents, for those with gaps by a stride of zero and
    by their first and last elements (views may lie in each other's gaps)."""
    spans = []
    for t in tensors:
        start, size = t.data_ptr(), t.element_size()
        if t.is_contiguous() or _dense(t):
            spans.append((start, start + t.numel() * size))
        elif any(st == 0 and n > 1 for st, n in zip(t.stride(), t.shape)):
            return True
        else:
            last = start + size * sum(st * (n - 1) for st, n in zip(t.stride(), t.shape))
            spans += [(start, start + size), (last, last + size)]
    spans.sort()
    return any(b[0] < a[1] for a, b in zip(spans, spans[1:]))


def _run(grads, max_norm: float, eps: float, scale: bool) -> torch.Tensor:
    if isinstance(grads, torch.Tensor):
        grads = [grads]
    grads = list(grads)
    fast = _fast()
    if fast is not None:
        norm = fast.clip(grads, max_norm, eps, scale)
        if norm is not None:
            return norm
    if not grads:
        raise ValueError("no tensors given")
    for i, t in enumerate(grads):
        if not isinstance(t, torch.Tensor):
            raise ValueError(f"tensor {i} is a {type(t).__name__}")
        if t.device.type != "cuda":
            raise RuntimeError(f"orthossm_amd runs on a ROCm GPU only; tensor {i} is on {t.device}")
        if t.device != grads[0].device:
            raise ValueError(f"tensor {i} is on {t.device}, the first on {grads[0].device}")
        if t.dtype not in (torch.float32, torch.bfloat16):
            raise TypeError(f"tensor {i} is {t.dtype}; use float32 or bfloat16")
        if scale and t.requires_grad:
            raise ValueError(f"tensor {i} requires a gradient; give the gradients")
    # (a tensor with gaps in memory is worked on in a copy)
    work = [t if t.is_contiguous() or _dense(t) else t.contiguous() for t in grads]
    if scale and _share_memory([t for t in grads if t.numel()]):
        raise ValueError("a tensor is given twice, or two share memory")
    lib = nat.load()
    dev, n = grads[0].device, len(work)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    a = nat.ClipArgs()
    a.abi_version, a.flags, a.count = nat.ABI_VERSION, nat.CLIP_SCALE if scale else 0, n
    a.tensors = (ctypes.c_void_p * n)(*(t.data_ptr() for t in work))
    a.sizes = (ctypes.c_int64 * n)(*(t.numel() for t in work))
    a.dtypes = (ctypes.c_int32 * n)(*(_dtype_code(t.dtype) for t in work))
    a.max_norm, a.eps, a.norm = float(max_norm), float(eps), norm.data_ptr()
    ws = _scratch(lib.osm_clip_workspace_bytes(ctypes.byref(a)), dev)
    with on_device(dev):
        nat.check(lib.osm_clip_grad_norm(ctypes.byref(a), ctypes.c_void_p(ws.data_ptr()), ws.numel(),
                                         ctypes.c_void_p(_current_stream(dev))))
    if scale:
        for t, w in zip(grads, work):
            if w is t:
                written(t)
            else:
                t.copy_(w)
    return norm


def grad_norm(grads: Iterable[torch.Tensor] | torch.Tensor) -> torch.Tensor:
    """The 2-norm over all elements of all tensors, a 0-d fp32 device tensor."""
    return _run(grads, 0.0, 0.0, False)


def clip_grad_norm(grads: Iterable[torch.Tensor] | torch.Tensor, max_norm: float, *, eps: float = 1e-6) -> torch.Tensor:
    """Scales the gradients in place to a norm of at most about ``max_norm``
    (by min(1, max_norm / (norm + eps))) and returns the norm they had, a 0-d
    fp32 device tensor."""
    return _run(grads, max_norm, eps, True)
