"""Sequences of one token through the chunked forward and the backward, with
token strides below a row's length: that stride of a single token is any number.
Tolerances as in test_gpu_delta.py."""
import pytest
import torch

from oracle import delta as O
from orthossm_amd import gated_delta
from test_gpu_delta import BF16, FP32, args, close, make

pytestmark = pytest.mark.gpu


def tokens_last(t, dev):
    """[B,1,heads,size] in memory as [B,heads,size,1]."""
    B, S, heads, size = t.shape
    return torch.empty(B, heads, size, S, dtype=t.dtype, device=dev).copy_(t.permute(0, 2, 3, 1))


def as_rows(t):
    """[B,heads,size,1] as a view [B,1,heads,size]: strides (heads size, 1, size, 1)."""
    t = t.permute(0, 3, 1, 2)
    assert t.stride(1) == 1
    return t


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,Hk,dk,dv", [(2, 2, 16, 16), (4, 2, 50, 33), (2, 1, 128, 128), (1, 1, 64, 1)])
def test_token_last_layout(dev, H, Hk, dk, dv, dtype):
    t = make(3, 1, H, dk, dv, Hk, dtype, seed=dk)
    want = O.gated_delta_grads(*args(t), t["grad_out"], t["grad_state"], state_init=t["state_init"])
    leaves = [as_rows(tokens_last(t[n], dev)).requires_grad_() for n in ("q", "k", "v")]
    leaves += [t[n].to(dev).requires_grad_() for n in ("g", "beta", "state_init")]
    out, fin = gated_delta(*leaves[:5], state_init=leaves[5], return_state=True)
    grads = torch.autograd.grad((out.permute(0, 2, 3, 1), fin), leaves,
                                (tokens_last(t["grad_out"], dev), t["grad_state"].to(dev)))
    names = ("out", "state", "grad_q", "grad_k", "grad_v", "grad_g", "grad_beta", "grad_init")
    for name, got, ref in zip(names, (out, fin, *grads), want):
        tol = BF16 if got.dtype == torch.bfloat16 else 2 * FP32 if name in ("grad_g", "grad_beta") else FP32
        close(got.detach(), ref, tol, name)


def test_broadcast_gradient_of_one_value(dev):
    """out.sum(): a gradient with every stride zero, rows of one element."""
    t = make(2, 1, 2, 16, 1)
    t["grad_out"] = torch.ones_like(t["grad_out"])
    want = O.gated_delta_grads(*args(t), t["grad_out"], None, state_init=t["state_init"])[2:]
    leaves = [as_rows(tokens_last(t[n], dev)).requires_grad_() for n in ("q", "k", "v")]
    leaves += [t[n].to(dev).requires_grad_() for n in ("g", "beta", "state_init")]
    out = gated_delta(*leaves[:5], state_init=leaves[5])
    for i, (got, ref) in enumerate(zip(torch.autograd.grad(out.sum(), leaves), want)):
        close(got, ref, 2 * FP32 if i in (3, 4) else FP32, i)


@pytest.mark.parametrize("grad", [False, True])
def test_token_stride_past_the_limit(dev, grad):
    """Time-major tensors of one token: a stride that no chunk could have."""
    t = {n: x.to(dev) for n, x in make(2, 1, 2, 16).items()}
    far = [x.as_strided(x.shape, (x.stride(0), 1 << 23, *x.stride()[2:])) for x in args(t)]
    near, far = ([x.detach().requires_grad_(grad) for x in ins] for ins in (args(t), far))
    want, got = (gated_delta(*ins, state_init=t["state_init"], return_state=True) for ins in (near, far))
    assert all(torch.equal(x, y) for x, y in zip(want, got))
    if grad:
        go = t["grad_out"].as_strided(t["grad_out"].shape, (32, 1 << 23, 16, 1))
        for x, y in zip(torch.autograd.grad(want[0], near, t["grad_out"]), torch.autograd.grad(got[0], far, go)):
            assert torch.equal(x, y)
