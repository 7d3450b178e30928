"""The EMA with a learned gate over the C ABI (HIP kernels on gfx950).

Per batch row and channel, with a gate of its own for every token:

    h_t = a_t h_{t-1} + (1 - a_t) x_t,   a_t = sigmoid(gate_t)

``gated_ema``           the differentiable op: gradients to x, the gate and the
                        initial state.
``gated_ema_forward``   the forward alone.
``gated_ema_backward``  the three gradients from dL/dh (+ dL/d final state).
``gated_ema_step``      one token a row, the states updated in place in a pool
                        (serving).

x and gate [B,S,D] fp32 or bf16 (mixed or other types go to fp32), states [B,D]
fp32, h in x's type.  ``lengths`` [B]: tokens in use of each row; those at and
past it are not read, leave the state as it is and give zeros, outputs and
gradients alike.

All run on the current torch stream of the inputs' device and never
synchronise the host.  There is no CPU path.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _native as nat
from . import ops
from .delta import _dest, _extent, _lengths, _scratch, _state, apart, differentiable, on_device, written
from .ops import _after_launch, _current_stream, _dtype_code, _fast


def _extension():
    """The native launch path, which carries no test aids."""
    return None if ops._poll_limit_zero else _fast()


def _set_seq(r: nat.Seq, t: torch.Tensor) -> None:
    """[B,S,D], or [B,D] (one token)."""
    r.p, r.stride_b, r.stride_s = t.data_ptr(), t.stride(0), t.stride(1) if t.dim() == 3 else 0


def _unit(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _check(x, gate, dims: int, form: str):
    for name, t in (("x", x), ("gate", gate)):
        if not isinstance(t, torch.Tensor) or t.dim() != dims or t.shape[-1] < 1:
            raise ValueError(f"{name} must be a {form} tensor with D >= 1")
        if t.device.type != "cuda":
            raise RuntimeError(f"orthossm_amd runs on a ROCm GPU only; {name} is on {t.device}")
    if gate.shape != x.shape or gate.device != x.device:
        raise ValueError(f"gate {tuple(gate.shape)} on {gate.device} does not match x {tuple(x.shape)} on {x.device}")
    if not (x.dtype == gate.dtype and x.dtype in (torch.float32, torch.bfloat16)):
        x, gate = x.float(), gate.float()
    return _unit(x), _unit(gate)


def _prepare(x, gate, state_init, lengths):
    x, gate = _check(x, gate, 3, "[B,S,D]")
    dev = x.device
    B, S, D = x.shape
    init = _state(state_init, (B, D), dev, "state_init")
    lens = _lengths(lengths, B, S, dev)
    a = nat.EmaArgs()
    a.abi_version = nat.ABI_VERSION
    a.dtype = _dtype_code(x.dtype) | (nat.FLAG_POLL_LIMIT_ZERO if ops._poll_limit_zero else 0)
    a.B, a.S, a.D = B, S, D
    _set_seq(a.x, x)
    _set_seq(a.gate, gate)
    a.lengths = lens.data_ptr() if lens is not None else None
    a.state_init = init.data_ptr() if init is not None else None
    return a, (x, gate, init, lens)


def _forward(x, gate, state_init, lengths, out, return_state, state_out, save):
    lib = nat.load()
    a, keep = _prepare(x, gate, state_init, lengths)
    x, given = keep[0], (out, state_out)
    dev, state = x.device, (a.B, a.D)
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=dev)
    else:
        _dest(out, x.shape, x.dtype, dev, "out")
    _set_seq(a.out, out)
    if state_out is not None:
        _dest(state_out, state, torch.float32, dev, "state_out")
    elif return_state:
        state_out = torch.empty(state, dtype=torch.float32, device=dev)
    ins = dict(zip(("x", "gate", "state_init", "lengths"), keep))
    if given[0] is not None:
        apart("out", out, {**ins, "state_out": state_out})
    if given[1] is not None:
        apart("state_out", state_out, ins, "state_init")
    a.state_out = state_out.data_ptr() if state_out is not None else None
    saved = None
    if save:
        saved = _scratch(lib.osm_gated_ema_saved_bytes(ctypes.byref(a)), dev)
        a.saved = saved.data_ptr()
    ws = _scratch(lib.osm_gated_ema_workspace_bytes(ctypes.byref(a)), dev)
    with on_device(dev):
        stream = _current_stream(dev)
        nat.check(lib.osm_gated_ema_fwd(ctypes.byref(a), ctypes.c_void_p(ws.data_ptr()), ws.numel(), ctypes.c_void_p(stream)))
        if ws.numel():
            _after_launch(ws, stream, "gated_ema_forward")
    written(*given)
    return out, state_out, saved, keep


def gated_ema_forward(x: torch.Tensor, gate: torch.Tensor, *, state_init: torch.Tensor | None = None,
                      lengths: torch.Tensor | None = None, out: torch.Tensor | None = None, return_state: bool = False,
                      state_out: torch.Tensor | None = None):
    """The gated EMA over sequences.  ``state_init`` is zeros by default.
    Returns h [B,S,D] in x's type, and the state after the last token [B,D]
    fp32 when ``return_state``.  ``out`` and ``state_out`` (contiguous; state_out
    may be state_init, else they lie in no argument's memory) receive the results
    instead of new tensors."""
    fast = _extension()
    if fast is not None and out is None and state_out is None:
        res = fast.ema_forward(x, gate, lengths, state_init, return_state)
        if res is not None:
            return res if return_state else res[0]
    out, fin, _, _ = _forward(x, gate, state_init, lengths, out, return_state, state_out, False)
    return (out, fin) if return_state else out


def _backward(x, gate, lengths, saved, grad_out, grad_state, need_init: bool):
    """The three gradients; ``saved`` as _forward gave it."""
    lib = nat.load()
    a, keep = _prepare(x, gate, None, lengths)
    x, gate = keep[:2]
    dev = x.device
    if not isinstance(grad_out, torch.Tensor) or grad_out.shape != x.shape:
        raise ValueError(f"grad_out must be a tensor of shape {tuple(x.shape)}")
    go = _unit(grad_out.to(device=dev, dtype=x.dtype))
    gs = _state(grad_state, (a.B, a.D), dev, "grad_state")
    gx, gg = (torch.empty(x.shape, dtype=x.dtype, device=dev) for _ in range(2))
    gi = torch.empty((a.B, a.D), dtype=torch.float32, device=dev) if need_init else None
    if saved.dtype != torch.uint8 or saved.device != dev or not saved.is_contiguous() or \
            saved.numel() != lib.osm_gated_ema_saved_bytes(ctypes.byref(a)):
        raise RuntimeError("a saved tensor came back in another form: gated_ema")
    a.saved = saved.data_ptr()
    b = nat.EmaBwdArgs()
    for name, t in (("grad_out", go), ("grad_x", gx), ("grad_gate", gg)):
        _set_seq(getattr(b, name), t)
    b.grad_state = gs.data_ptr() if gs is not None else None
    b.grad_init = gi.data_ptr() if gi is not None else None
    ws = _scratch(lib.osm_gated_ema_bwd_workspace_bytes(ctypes.byref(a)), dev)
    with on_device(dev):
        stream = _current_stream(dev)
        nat.check(lib.osm_gated_ema_bwd(ctypes.byref(a), ctypes.byref(b), ctypes.c_void_p(ws.data_ptr()), ws.numel(),
                                        ctypes.c_void_p(stream)))
        if ws.numel():
            _after_launch(ws, stream, "gated_ema_backward")
    return gx, gg, gi


def gated_ema_backward(x: torch.Tensor, gate: torch.Tensor, grad_out: torch.Tensor, *,
                       state_init: torch.Tensor | None = None, lengths: torch.Tensor | None = None,
                       grad_state: torch.Tensor | None = None, need_init: bool = False):
    """Backward of ``gated_ema_forward`` from its inputs, ``grad_out`` = dL/dh
    and ``grad_state`` = dL/d final state or None.  Runs the forward again for
    the states along the sequence (``gated_ema`` keeps them instead).  Returns
    (grad_x, grad_gate in the inputs' type, grad_init fp32 or None)."""
    _, _, saved, keep = _forward(x, gate, state_init, lengths, None, False, None, True)
    return _backward(keep[0], keep[1], keep[3], saved, grad_out, grad_state, need_init)


class _GatedEmaFunction(torch.autograd.Function):
    """Saves the inputs and the states along the sequence."""

    @staticmethod
    def forward(ctx, x, gate, state_init, lengths):
        ctx.set_materialize_grads(False)   # an unused output's gradient stays None
        out, fin, saved, keep = _forward(x, gate, state_init, lengths, None, True, None, True)
        ctx.save_for_backward(keep[0], keep[1], keep[3], saved)
        ctx.types = [None if t is None else t.dtype for t in (x, gate, state_init)]
        return out, fin

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out, grad_state):
        x, gate, lengths, saved = ctx.saved_tensors
        if grad_out is None:
            grad_out = torch.zeros_like(x)
        need = ctx.needs_input_grad
        grads = _backward(x, gate, lengths, saved, grad_out, grad_state, need[2])
        return (*(t.to(dt) if n else None for t, dt, n in zip(grads, ctx.types, need)), None)


def gated_ema(x: torch.Tensor, gate: torch.Tensor, *, state_init: torch.Tensor | None = None,
              lengths: torch.Tensor | None = None, return_state: bool = False):
    """``gated_ema_forward`` as a differentiable op: gradients flow to x, gate
    and state_init, from the output and the final state.  Returns h, or (h,
    final state) when ``return_state``."""
    fast = _extension()
    if fast is not None:
        res = fast.gated_ema(x, gate, lengths, state_init)
        if res is not None:
            return res if return_state else res[0]
    if differentiable(x, gate, state_init):
        out, fin = _GatedEmaFunction.apply(x, gate, state_init, lengths)
        return (out, fin) if return_state else out
    return gated_ema_forward(x, gate, state_init=state_init, lengths=lengths, return_state=return_state)


def _reads_states(t: torch.Tensor, state: torch.Tensor, slots) -> bool:
    """Whether a row of ``t`` [B,D] lies where another row's state is written (its
    own, at the same place in both, it reads before)."""
    (a, b), (c, d) = _extent(t), _extent(state)
    if not t.numel() or not state.numel() or a >= d or c >= b:
        return False
    step, rows = t.stride(0) * t.element_size() if t.shape[0] > 1 else 0, state.stride(0) * 4
    if slots is None and a == c and t.dtype == state.dtype and (step == rows or t.shape[0] == 1):
        return False
    # beside the states: in the gaps between them, at whole times their distance
    gap = (a - c) % rows
    return step % rows != 0 or gap < 4 * state.shape[1] or gap + t.shape[1] * t.element_size() > rows


def gated_ema_step(x: torch.Tensor, gate: torch.Tensor, state: torch.Tensor, *, slots: torch.Tensor | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """One token a row: x, gate [B,D], and the states [slots,D] fp32, which are
    updated in place.  Row b's state is slot b, or ``slots[b]`` (int64, on the
    device, no slot twice): a negative one marks an idle row, whose output is 0;
    one past the pool gives NaN; neither touches a state.  x and gate lie in no
    state's memory (without slots they may be the states).  Returns h [B,D] in x's
    type, in ``out`` (contiguous, in no argument's memory) if given."""
    fast = _extension()
    if fast is not None and out is None:
        res = fast.ema_step(x, gate, state, slots)
        if res is not None:
            return res
    lib = nat.load()
    x, gate = _check(x, gate, 2, "[B,D]")
    dev = x.device
    B, D = x.shape
    if not isinstance(state, torch.Tensor) or state.dim() != 2 or state.shape[1] != D or state.dtype != torch.float32 or \
            state.device != dev or not state[:1].is_contiguous() or state.stride(0) < D or state.requires_grad:
        raise ValueError(f"state must be a float32 tensor [slots,{D}] on {dev} without gradient, its slots contiguous")
    if slots is None:
        if state.shape[0] < B:
            raise ValueError(f"state has {state.shape[0]} slots for {B} rows")
    elif not isinstance(slots, torch.Tensor) or tuple(slots.shape) != (B,) or slots.dtype != torch.int64 or \
            slots.device != dev or not slots.is_contiguous():
        raise ValueError(f"slots must be a contiguous int64 tensor of shape ({B},) on {dev}")
    for name, t in (("x", x), ("gate", gate)):
        if _reads_states(t, state, slots):
            raise ValueError(f"{name} shares memory with state")
    given = out
    if out is None:
        out = torch.empty((B, D), dtype=x.dtype, device=dev)
    else:
        _dest(out, (B, D), x.dtype, dev, "out")
        apart("out", out, dict(x=x, gate=gate, state=state, slots=slots))
    a = nat.EmaStepArgs()
    a.abi_version, a.dtype = nat.ABI_VERSION, _dtype_code(x.dtype)
    a.B, a.D = B, D
    for name, t in (("x", x), ("gate", gate), ("out", out)):
        _set_seq(getattr(a, name), t)
    a.state, a.state_stride, a.n_slots = state.data_ptr(), state.stride(0), state.shape[0]
    a.slots = slots.data_ptr() if slots is not None else None
    with on_device(dev):
        nat.check(lib.osm_gated_ema_step(ctypes.byref(a), ctypes.c_void_p(_current_stream(dev))))
    written(state, given)
    return out
