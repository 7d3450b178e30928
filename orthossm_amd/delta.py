"""The gated delta rule over the C ABI (HIP kernels on gfx950).

Per batch row and head a matrix state S [dk, dv], one step of gradient descent
on |S^T k - v|^2 a token, at rate beta, after a decay e^g:

    S_t = e^{g_t} S_{t-1} + k_t u_t^T,   u_t = beta_t (v_t - e^{g_t} S_{t-1}^T k_t)
    o_t = scale S_t^T q_t

``gated_delta``           the differentiable op: gradients to q, k, v, g, beta
                          and the initial state.
``gated_delta_forward``   the forward alone.
``gated_delta_backward``  the six gradients from dL/do (+ dL/d final state).
``gated_delta_step``      one token a row, the states updated in place in a
                          pool (serving).

q, k [B,S,Hk,dk] and v [B,S,H,dv] fp32 or bf16 (mixed or other types go to
fp32), H a multiple of Hk (head h uses q/k head h // (H // Hk)), dk up to 128;
g (the logarithm of the decay) and beta [B,S,H] fp32; states [B,H,dk,dv] fp32.
``lengths`` [B]: tokens in use of each row; those at and past it are not read,
leave the state as it is and give zeros, outputs and gradients alike.

All run on the current torch stream of the inputs' device and never
synchronise the host.  There is no CPU path.
"""
from __future__ import annotations

import contextlib
import ctypes

import torch
from torch.autograd.forward_ad import unpack_dual
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from . import _native as nat
from .ops import _current_device, _current_stream, _dtype_code, _fast


def on_device(dev: torch.device):
    """Makes ``dev`` current for a launch, where it is not already."""
    return contextlib.nullcontext() if dev.index == _current_device() else torch.cuda.device(dev)


def _set_rows(r: nat.Rows, t: torch.Tensor) -> None:
    """[B,S,H,d] or [B,S,H] (one element a head)."""
    r.p, r.stride_b, r.stride_s, r.stride_h = t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)


def _unit_rows(t: torch.Tensor) -> torch.Tensor:
    near = t.dim() < 4 or t.shape[1] <= 1 or t.shape[3] <= t.stride(1) <= nat.DELTA_MAX_STRIDE
    return t if near and (t.stride(-1) == 1 or t.shape[-1] == 1) else t.contiguous()


def differentiable(*tensors) -> bool:
    """Whether a call on these has a derivative to record, or (a dual number of
    forward-mode differentiation) one that its autograd function refuses."""
    ts = [t for t in tensors if isinstance(t, torch.Tensor)]
    return (torch.is_grad_enabled() and any(t.requires_grad for t in ts)) or \
        any(unpack_dual(t).tangent is not None for t in ts)


def _check_qkv(q, k, v, dims: int, form: str):
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor) or t.dim() != dims:
            raise ValueError(f"{name} must be a {form} tensor")
        if t.device.type != "cuda":
            raise RuntimeError(f"orthossm_amd runs on a ROCm GPU only; {name} is on {t.device}")
        if t.device != q.device:
            raise ValueError(f"{name} is on {t.device}, q on {q.device}")
    if k.shape != q.shape or v.shape[:-2] != q.shape[:-2]:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not match")
    Hk, dk, H, dv = q.shape[-2], q.shape[-1], v.shape[-2], v.shape[-1]
    if Hk < 1 or H < 1 or H % Hk:
        raise ValueError(f"v's heads ({H}) must be a multiple of q's and k's ({Hk})")
    if not 1 <= dk <= nat.DELTA_MAX_DK or dv < 1:
        raise ValueError(f"head sizes must be at least 1, and dk at most {nat.DELTA_MAX_DK} (dk={dk}, dv={dv})")
    if not (q.dtype == k.dtype == v.dtype and q.dtype in (torch.float32, torch.bfloat16)):
        q, k, v = q.float(), k.float(), v.float()
    return _unit_rows(q), _unit_rows(k), _unit_rows(v)


def _gate(t, shape, dev, name: str) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be a tensor of shape {tuple(shape)}")
    t = t.to(device=dev, dtype=torch.float32)
    return t if t.dim() < 3 or t.shape[1] <= 1 or t.stride(1) <= nat.DELTA_MAX_STRIDE else t.contiguous()


def _state(t, shape, dev, name: str) -> torch.Tensor | None:
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be a tensor of shape {tuple(shape)}")
    return t.to(device=dev, dtype=torch.float32).contiguous()


def _dest(t, shape, dtype, dev, name: str) -> None:
    if not isinstance(t, torch.Tensor) or tuple(t.shape) != tuple(shape) or t.dtype != dtype or t.device != dev or \
            not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)} on {dev}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient, which what is written into it has not")


def _extent(t: torch.Tensor) -> tuple[int, int]:
    """First byte of t's elements and the one after the last."""
    last = sum(st * (n - 1) for st, n in zip(t.stride(), t.shape))
    return t.data_ptr(), t.data_ptr() + t.element_size() * (1 + last)


def apart(name: str, t: torch.Tensor, others: dict, may_be: str | None = None) -> None:
    """Refuses an output ``t`` that lies in the memory of another argument, which
    some of a launch's workgroups would read after others wrote it.  It may be
    the one named ``may_be``, as a whole."""
    for other, o in others.items():
        if o is None or o is t and other == may_be or not o.numel() or not t.numel():
            continue
        (a, b), (c, d) = _extent(t), _extent(o)
        whole = other == may_be and a == c and o.dtype == t.dtype and o.shape == t.shape and o.is_contiguous()
        if not whole and a < d and c < b:
            raise ValueError(f"{name} shares memory with {other}")


def written(*tensors) -> None:
    """Tells autograd that a launch wrote into these (None: skipped): a graph
    that saved one refuses its backward, as after torch's own in-place
    operations."""
    for t in tensors:
        if t is not None and not t.is_inference():
            increment_version(t)


def _lengths(t, B: int, S: int, dev) -> torch.Tensor | None:
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or tuple(t.shape) != (B,) or t.is_floating_point() or t.is_complex() or \
            t.dtype == torch.bool:
        raise ValueError(f"lengths must be a whole-number tensor of shape ({B},)")
    if t.dtype is not torch.int32:
        t = t.to(torch.int64).clamp(0, S)       # (in its own type S may not fit)
    return t.to(device=dev, dtype=torch.int32).contiguous()


def _prepare(q, k, v, g, beta, scale, state_init, lengths):
    q, k, v = _check_qkv(q, k, v, 4, "[B,S,heads,size]")
    dev = q.device
    B, S, Hk, dk = q.shape
    H, dv = v.shape[2:]
    g, beta = _gate(g, (B, S, H), dev, "g"), _gate(beta, (B, S, H), dev, "beta")
    init = _state(state_init, (B, H, dk, dv), dev, "state_init")
    lens = _lengths(lengths, B, S, dev)
    a = nat.DeltaArgs()
    a.abi_version, a.dtype = nat.ABI_VERSION, _dtype_code(q.dtype)
    a.B, a.S, a.H, a.Hk, a.dk, a.dv = B, S, H, Hk, dk, dv
    a.scale = dk ** -0.5 if scale is None else float(scale)
    for name, t in (("q", q), ("k", k), ("v", v), ("g", g), ("beta", beta)):
        _set_rows(getattr(a, name), t)
    a.lengths = lens.data_ptr() if lens is not None else None
    a.state_init = init.data_ptr() if init is not None else None
    return a, (q, k, v, g, beta, init, lens)


def _scratch(nbytes: int, dev) -> torch.Tensor:
    return torch.empty(nbytes, dtype=torch.uint8, device=dev)


def _forward(q, k, v, g, beta, scale, state_init, lengths, out, return_state, state_out, save):
    fast = _fast()
    if fast is not None and out is None and state_out is None:
        res = fast.delta_forward(q, k, v, g, beta, scale, lengths, state_init, return_state, save)
        if res is not None:
            return (*res, (q, k, v, g, beta, state_init, lengths))
    lib = nat.load()
    a, keep = _prepare(q, k, v, g, beta, scale, state_init, lengths)
    v, given = keep[2], (out, state_out)
    dev, shape = v.device, (a.B, a.S, a.H, a.dv)
    if out is None:
        out = torch.empty(shape, dtype=v.dtype, device=dev)
    else:
        _dest(out, shape, v.dtype, dev, "out")
    _set_rows(a.out, out)
    state = (a.B, a.H, a.dk, a.dv)
    if state_out is not None:
        _dest(state_out, state, torch.float32, dev, "state_out")
    elif return_state:
        state_out = torch.empty(state, dtype=torch.float32, device=dev)
    ins = dict(zip(("q", "k", "v", "g", "beta", "state_init", "lengths"), keep))
    if given[0] is not None:
        apart("out", out, {**ins, "state_out": state_out}, "v")
    if given[1] is not None:
        apart("state_out", state_out, ins, "state_init")
    a.state_out = state_out.data_ptr() if state_out is not None else None
    saved = None
    if save:
        saved = _scratch(lib.osm_delta_saved_bytes(ctypes.byref(a)), dev)
        a.saved = saved.data_ptr()
    ws = _scratch(lib.osm_delta_workspace_bytes(ctypes.byref(a)), dev)
    with on_device(dev):
        nat.check(lib.osm_delta_fwd(ctypes.byref(a), ctypes.c_void_p(ws.data_ptr()), ws.numel(),
                                    ctypes.c_void_p(_current_stream(dev))))
    written(*given)
    return out, state_out, saved, keep


def gated_delta_forward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor, *,
                        scale: float | None = None, state_init: torch.Tensor | None = None,
                        lengths: torch.Tensor | None = None, out: torch.Tensor | None = None,
                        return_state: bool = False, state_out: torch.Tensor | None = None):
    """The gated delta rule over sequences.  ``scale`` is 1/sqrt(dk) by
    default, ``state_init`` zeros.  Returns out [B,S,H,dv] in v's type, and
    the state after the last token [B,H,dk,dv] fp32 when ``return_state``.
    ``out`` and ``state_out`` (contiguous; out may be v and state_out state_init,
    else they lie in no argument's memory) receive the results instead of new
    tensors."""
    out, fin, _, _ = _forward(q, k, v, g, beta, scale, state_init, lengths, out, return_state, state_out, False)
    return (out, fin) if return_state else out


def _backward(inputs, scale, lengths, saved, grad_out, grad_state, need_init: bool):
    """The six gradients; ``inputs`` (q, k, v, g, beta), ``lengths`` and
    ``saved`` as _forward gave them."""
    fast = _fast()
    if fast is not None:
        res = fast.delta_backward(*inputs, scale, lengths, saved, grad_out, grad_state, need_init)
        if res is not None:
            return res
    lib = nat.load()
    a, keep = _prepare(*inputs, scale, None, lengths)
    q, k, v, g = keep[:4]
    dev = v.device
    if not isinstance(grad_out, torch.Tensor) or grad_out.shape != v.shape:
        raise ValueError(f"grad_out must be a tensor of shape {tuple(v.shape)}")
    go = _unit_rows(grad_out.to(device=dev, dtype=v.dtype))
    gs = _state(grad_state, (a.B, a.H, a.dk, a.dv), dev, "grad_state")
    gq, gk, gv = (torch.empty(t.shape, dtype=t.dtype, device=dev) for t in (q, k, v))
    gg, gb = (torch.empty(g.shape, dtype=torch.float32, device=dev) for _ in range(2))
    gi = torch.empty((a.B, a.H, a.dk, a.dv), dtype=torch.float32, device=dev) if need_init else None
    if saved.dtype != torch.uint8 or saved.device != dev or not saved.is_contiguous() or \
            saved.numel() != lib.osm_delta_saved_bytes(ctypes.byref(a)):
        raise RuntimeError("a saved tensor came back in another form: gated_delta")
    a.saved = saved.data_ptr()
    b = nat.DeltaBwdArgs()
    for name, t in (("grad_out", go), ("grad_q", gq), ("grad_k", gk), ("grad_v", gv), ("grad_g", gg),
                    ("grad_beta", gb)):
        _set_rows(getattr(b, name), t)
    b.grad_state = gs.data_ptr() if gs is not None else None
    b.grad_init = gi.data_ptr() if gi is not None else None
    ws = _scratch(lib.osm_delta_bwd_workspace_bytes(ctypes.byref(a)), dev)
    with on_device(dev):
        nat.check(lib.osm_delta_bwd(ctypes.byref(a), ctypes.byref(b), ctypes.c_void_p(ws.data_ptr()), ws.numel(),
                                    ctypes.c_void_p(_current_stream(dev))))
    return gq, gk, gv, gg, gb, gi


def gated_delta_backward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                         grad_out: torch.Tensor, *, scale: float | None = None,
                         state_init: torch.Tensor | None = None, lengths: torch.Tensor | None = None,
                         grad_state: torch.Tensor | None = None, need_init: bool = False):
    """Backward of ``gated_delta_forward`` from its inputs, ``grad_out`` =
    dL/dout and ``grad_state`` = dL/d final state or None.  Runs the forward
    again for what it needs of it (``gated_delta`` keeps that instead).
    Returns (grad_q, grad_k, grad_v in the inputs' type, grad_g, grad_beta
    fp32, grad_init fp32 or None)."""
    _, _, saved, keep = _forward(q, k, v, g, beta, scale, state_init, lengths, None, False, None, True)
    return _backward(keep[:5], scale, keep[6], saved, grad_out, grad_state, need_init)


class _GatedDeltaFunction(torch.autograd.Function):
    """Saves the inputs, the chunks' triangular systems and start states."""

    @staticmethod
    def forward(ctx, q, k, v, g, beta, state_init, lengths, scale):
        ctx.set_materialize_grads(False)   # an unused output's gradient stays None
        out, fin, saved, keep = _forward(q, k, v, g, beta, scale, state_init, lengths, None, True, None, True)
        ctx.save_for_backward(*keep[:5], keep[6], saved)
        ctx.scale = scale
        ctx.types = [t.dtype for t in (q, k, v, g, beta)] + [None if state_init is None else state_init.dtype]
        return out, fin

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out, grad_state):
        *inputs, lengths, saved = ctx.saved_tensors
        if grad_out is None:
            grad_out = torch.zeros_like(inputs[2])
        need = ctx.needs_input_grad
        grads = _backward(inputs, ctx.scale, lengths, saved, grad_out, grad_state, need[5])
        return (*(t.to(dt) if n else None for t, dt, n in zip(grads, ctx.types, need)), None, None)


def gated_delta(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor, *,
                scale: float | None = None, state_init: torch.Tensor | None = None,
                lengths: torch.Tensor | None = None, return_state: bool = False):
    """``gated_delta_forward`` as a differentiable op: gradients flow to q, k,
    v, g, beta and state_init, from the output and the final state.  Returns
    out, or (out, final state) when ``return_state``."""
    fast = _fast()
    if fast is not None:
        res = fast.gated_delta(q, k, v, g, beta, scale, lengths, state_init, return_state)
        if res is not None:
            return res if return_state else res[0]
    if differentiable(q, k, v, g, beta, state_init):
        out, fin = _GatedDeltaFunction.apply(q, k, v, g, beta, state_init, lengths, scale)
        return (out, fin) if return_state else out
    return gated_delta_forward(q, k, v, g, beta, scale=scale, state_init=state_init, lengths=lengths,
                               return_state=return_state)


def gated_delta_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                     state: torch.Tensor, *, scale: float | None = None, slots: torch.Tensor | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """One token a row: q, k [B,Hk,dk], v [B,H,dv], g, beta [B,H], and the
    states [slots,H,dk,dv] fp32, which are updated in place.  Row b's state is
    slot b, or ``slots[b]`` (int64, on the device, no slot twice): a negative
    one marks an idle row, whose output is 0; one past the pool gives NaN;
    neither touches a state.  Returns out [B,H,dv] in v's type, in ``out``
    (contiguous; may be v, else in no argument's memory) if given."""
    fast = _fast()
    if fast is not None and out is None:
        res = fast.delta_step(q, k, v, g, beta, state, scale, slots)
        if res is not None:
            return res
    lib = nat.load()
    q, k, v = _check_qkv(q, k, v, 3, "[B,heads,size]")
    dev = q.device
    B, Hk, dk = q.shape
    H, dv = v.shape[1:]
    g, beta = _gate(g, (B, H), dev, "g"), _gate(beta, (B, H), dev, "beta")
    if not isinstance(state, torch.Tensor) or state.dim() != 4 or tuple(state.shape[1:]) != (H, dk, dv) or \
            state.dtype != torch.float32 or state.device != dev or not state[:1].is_contiguous() or \
            state.stride(0) < H * dk * dv or state.requires_grad:
        raise ValueError(f"state must be a float32 tensor [slots,{H},{dk},{dv}] on {dev} without gradient, its slots "
                         "contiguous")
    if slots is None:
        if state.shape[0] < B:
            raise ValueError(f"state has {state.shape[0]} slots for {B} rows")
    elif not isinstance(slots, torch.Tensor) or tuple(slots.shape) != (B,) or slots.dtype != torch.int64 or \
            slots.device != dev or not slots.is_contiguous():
        raise ValueError(f"slots must be a contiguous int64 tensor of shape ({B},) on {dev}")
    given = out
    if out is None:
        out = torch.empty((B, H, dv), dtype=v.dtype, device=dev)
    else:
        _dest(out, (B, H, dv), v.dtype, dev, "out")
        apart("out", out, dict(q=q, k=k, v=v, g=g, beta=beta, state=state, slots=slots), "v")
    a = nat.DeltaStepArgs()
    a.abi_version, a.dtype = nat.ABI_VERSION, _dtype_code(q.dtype)
    a.B, a.H, a.Hk, a.dk, a.dv = B, H, Hk, dk, dv
    a.scale = dk ** -0.5 if scale is None else float(scale)
    for name, t in (("q", q), ("k", k), ("v", v), ("out", out), ("g", g), ("beta", beta)):
        r = getattr(a, name)
        r.p, r.stride_b, r.stride_s, r.stride_h = t.data_ptr(), t.stride(0), 0, t.stride(1)
    a.state, a.state_stride, a.n_slots = state.data_ptr(), state.stride(0), state.shape[0]
    a.slots = slots.data_ptr() if slots is not None else None
    with on_device(dev):
        nat.check(lib.osm_delta_step(ctypes.byref(a), ctypes.c_void_p(_current_stream(dev))))
    written(state, given)
    return out
