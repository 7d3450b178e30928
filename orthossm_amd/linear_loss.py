"""The cross entropy of a projection to a vocabulary over the C ABI (HIP kernels
on gfx950), without its logits.

    loss_n = log sum_v exp(hidden_n . weight_v) - hidden_n . weight_{targets_n}

``linear_cross_entropy``           the differentiable op: gradients to hidden
                                   and weight.
``linear_cross_entropy_forward``   (losses, lse) of every token.
``linear_cross_entropy_backward``  the two gradients from dL/d losses.

hidden [..., D] and weight [V,D] fp32 or bf16 (mixed or other types go to fp32)
with contiguous rows (others are copied first), targets whole numbers of
hidden's shape without D.  Tokens whose target is ``ignore_index`` count for
nothing, whatever their hidden rows hold: their losses and gradients are 0.  A
target outside [0, V) gives NaN: that token's loss, and every gradient that it
has a part in.  Infinities count as they are (a class whose weights are -inf is
left out where hidden is positive), but a logit of +inf makes NaN.  Logits, sums and losses are fp32; the gradients' factors
softmax - onehot are rounded to bf16 for bf16 inputs (up to 64 tokens: to the
sum of two bf16 numbers).

The backward forms the logits of a piece of the vocabulary at a time: its
memory is bounded by the pieces (302 MB of P, and as much of the weights where
they are copied: fp32, rows that are not whole units of 64 columns at multiples
of 16 bytes), not by the vocabulary.  All run on the current torch stream of
hidden's device and never synchronise the host.  There is no CPU path.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _native as nat
from .delta import _scratch, differentiable, on_device
from .norm import _matrix
from .ops import _current_stream, _dtype_code, _fast

_HOW = {"none": 0, "sum": 1, "mean": 2}


def _prepare(hidden, weight, targets, ignore_index):
    if not isinstance(hidden, torch.Tensor) or hidden.dim() < 1 or hidden.shape[-1] < 1:
        raise ValueError("hidden must be a [..., D] tensor with D >= 1")
    if hidden.device.type != "cuda":
        raise RuntimeError(f"orthossm_amd runs on a ROCm GPU only; hidden is on {hidden.device}")
    D, dev = hidden.shape[-1], hidden.device
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] != D or \
            weight.device != dev:
        raise ValueError(f"weight must be a [V,{D}] tensor on {dev} with V >= 1")
    if not isinstance(targets, torch.Tensor) or targets.shape != hidden.shape[:-1] or targets.is_floating_point() or \
            targets.is_complex() or targets.dtype == torch.bool or targets.device != dev:
        raise ValueError(f"targets must be a whole-number tensor of shape {tuple(hidden.shape[:-1])} on {dev}")
    if not (hidden.dtype == weight.dtype and hidden.dtype in (torch.float32, torch.bfloat16)):
        hidden, weight = hidden.float(), weight.float()
    targets = targets.to(torch.int64).contiguous()
    rows, w = _matrix(hidden), _matrix(weight)
    a = nat.LossArgs()
    a.abi_version, a.dtype = nat.ABI_VERSION, _dtype_code(hidden.dtype)
    a.N, a.D, a.V = rows.shape[0], D, weight.shape[0]
    a.hidden, a.hidden_stride = rows.data_ptr(), rows.stride(0)
    a.weight, a.weight_stride = w.data_ptr(), w.stride(0)
    a.targets, a.ignore_index = targets.data_ptr(), int(ignore_index)
    return a, (hidden, weight, targets), (rows, w)


def _forward(hidden, weight, targets, ignore_index, reduction="none"):
    """(losses, or their sum or mean; lse; the count that a mean divided by;
    the inputs as the kernels read them)."""
    lib = nat.load()
    a, ins, keep = _prepare(hidden, weight, targets, ignore_index)
    dev, shape = ins[0].device, ins[2].shape
    losses, lse = (torch.empty(shape, dtype=torch.float32, device=dev) for _ in range(2))
    a.losses, a.lse, loss, count = losses.data_ptr(), lse.data_ptr(), losses, None
    if reduction != "none":
        loss = torch.empty((), dtype=torch.float32, device=dev)
        a.loss = loss.data_ptr()
    if reduction == "mean":
        a.flags, count = nat.LOSS_MEAN, torch.empty((), dtype=torch.float32, device=dev)
        a.count = count.data_ptr()
    ws = _scratch(lib.osm_linear_ce_workspace_bytes(ctypes.byref(a)), dev)
    with on_device(dev):
        nat.check(lib.osm_linear_ce_fwd(ctypes.byref(a), ctypes.c_void_p(ws.data_ptr()), ws.numel(),
                                        ctypes.c_void_p(_current_stream(dev))))
    del keep
    return loss, lse, count, ins


def linear_cross_entropy_forward(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *,
                                 ignore_index: int = -100):
    """(losses, lse) fp32 of targets' shape: each token's loss and the logarithm
    of its sum of exponentials, 0 for tokens that do not count."""
    return _forward(hidden, weight, targets, ignore_index)[:2]


def _backward(hidden, weight, targets, lse, ignore_index, grad, count, grad_losses, need_hidden, need_weight):
    lib = nat.load()
    a, (hidden, weight, targets), keep = _prepare(hidden, weight, targets, ignore_index)
    dev = hidden.device
    if not isinstance(lse, torch.Tensor) or lse.shape != targets.shape or lse.dtype != torch.float32 or lse.device != dev:
        raise ValueError(f"lse must be a float32 tensor of shape {tuple(targets.shape)} on {dev}")
    lse = lse.contiguous()
    a.lse = lse.data_ptr()
    b = nat.LossBwdArgs()
    if grad is not None:
        grad = grad.to(device=dev, dtype=torch.float32).contiguous()
        b.grad = grad.data_ptr()
    if grad_losses is not None:
        if not isinstance(grad_losses, torch.Tensor) or grad_losses.shape != targets.shape:
            raise ValueError(f"grad_losses must be a tensor of shape {tuple(targets.shape)}")
        grad_losses = grad_losses.to(device=dev, dtype=torch.float32).contiguous()
        b.grad_losses = grad_losses.data_ptr()
    b.count = count.data_ptr() if count is not None else None
    gh = torch.empty(hidden.shape, dtype=hidden.dtype, device=dev) if need_hidden else None
    gw = torch.empty(weight.shape, dtype=weight.dtype, device=dev) if need_weight else None
    b.grad_hidden, b.grad_weight = (None if t is None else t.data_ptr() for t in (gh, gw))
    ws = _scratch(lib.osm_linear_ce_bwd_workspace_bytes(ctypes.byref(a)), dev)
    with on_device(dev):
        nat.check(lib.osm_linear_ce_bwd(ctypes.byref(a), ctypes.byref(b), ctypes.c_void_p(ws.data_ptr()), ws.numel(),
                                        ctypes.c_void_p(_current_stream(dev))))
    del keep
    return gh, gw


def linear_cross_entropy_backward(grad_losses: torch.Tensor, hidden: torch.Tensor, weight: torch.Tensor,
                                  targets: torch.Tensor, lse: torch.Tensor, *, ignore_index: int = -100,
                                  need_hidden: bool = True, need_weight: bool = True):
    """(grad_hidden, grad_weight) in the inputs' type, None for what is not
    needed, from dL/d losses and what the forward gave."""
    return _backward(hidden, weight, targets, lse, ignore_index, None, None, grad_losses, need_hidden, need_weight)


class _LinearCrossEntropyFunction(torch.autograd.Function):
    """Saves the inputs and lse (and the count of tokens): no logits."""

    @staticmethod
    def forward(ctx, hidden, weight, targets, ignore_index, reduction):
        loss, lse, count, ins = _forward(hidden, weight, targets, ignore_index, reduction)
        ctx.save_for_backward(*ins, lse, count)
        ctx.ignore_index, ctx.reduction, ctx.types = ignore_index, reduction, (hidden.dtype, weight.dtype)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        hidden, weight, targets, lse, count = ctx.saved_tensors
        each = ctx.reduction == "none"
        grads = _backward(hidden, weight, targets, lse, ctx.ignore_index, None if each else grad, count, grad if each else None,
                          *ctx.needs_input_grad[:2])
        return (*(None if t is None else t.to(dt) for t, dt in zip(grads, ctx.types)), None, None, None)


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *, ignore_index: int = -100,
                         reduction: str = "mean") -> torch.Tensor:
    """The cross entropy of softmax(hidden weight^T) against targets, fp32,
    differentiable in hidden and weight: the mean over the tokens that count (0
    where none does), their sum, or (``"none"``) every token's."""
    if reduction not in _HOW:
        raise ValueError(f"reduction must be 'mean', 'sum' or 'none', got {reduction!r}")
    fast = _fast()
    if fast is not None:
        loss = fast.linear_loss(hidden, weight, targets, ignore_index, _HOW[reduction])
        if loss is not None:
            return loss
    if differentiable(hidden, weight):
        return _LinearCrossEntropyFunction.apply(hidden, weight, targets, int(ignore_index), reduction)
    return _forward(hidden, weight, targets, ignore_index, reduction)[0]
