"""bf16 results of the gated delta rule are its fp32 results, rounded once.

bf16 inputs held as fp32 numbers go through the same kernels with the same
products: the second and third bf16 parts of such a number are zero, products
with them add exact zeros, and the others are added in the same order.  So the
output for bf16 inputs has to be the fp32 output of the same numbers, rounded,
bit for bit, and the states have to be equal.  An output from fewer parts
differs wherever what it leaves out moves a rounding.
"""
import pytest
import torch

from orthossm_amd import gated_delta_forward

pytestmark = pytest.mark.gpu


def make(dev, B, S, H, Hk, dk, dv, seed):
    gen = torch.Generator().manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=gen)

    q, k = (torch.nn.functional.normalize(rand(B, S, Hk, dk), dim=-1) for _ in range(2))
    t = dict(q=q.bfloat16(), k=k.bfloat16(), v=rand(B, S, H, dv).bfloat16(), g=-0.1 * torch.rand(B, S, H, generator=gen),
             beta=torch.sigmoid(rand(B, S, H)), state_init=0.5 * rand(B, H, dk, dv))
    return {n: x.to(dev) for n, x in t.items()}


def check(t):
    names = ("q", "k", "v", "g", "beta")
    out, fin = gated_delta_forward(*(t[n] for n in names), state_init=t["state_init"], return_state=True)
    wide, state = gated_delta_forward(*(t[n].float() for n in names), state_init=t["state_init"], return_state=True)
    assert out.dtype == torch.bfloat16 and wide.dtype == torch.float32
    assert torch.equal(fin, state)
    off = (out != wide.bfloat16()).float().mean().item()
    assert off == 0.0, f"{off:.1e} of the outputs differ from the fp32 ones, rounded"


# Whole rows and segments, head sizes of every number of blocks, on and off them.
SIZES = [(2, 150, 2, 2, 64, 64), (1, 200, 4, 2, 24, 40), (1, 130, 2, 1, 128, 128), (1, 140, 1, 1, 128, 40),
         (2, 100, 2, 2, 96, 200), (1, 70, 2, 2, 80, 33), (2, 9, 2, 1, 50, 50), (9, 300, 16, 16, 32, 16)]


@pytest.mark.parametrize("B,S,H,Hk,dk,dv", SIZES)
def test_forward(dev, B, S, H, Hk, dk, dv):
    check(make(dev, B, S, H, Hk, dk, dv, seed=dk + dv))


@pytest.mark.parametrize("B,S,H,Hk,dk,dv", SIZES)
def test_forward_with_cancellation(dev, B, S, H, Hk, dk, dv):
    """q = k and beta = 1: what is read of a start state a thousand times the
    values nearly cancels against what the updates take off it."""
    t = make(dev, B, S, H, Hk, dk, dv, seed=dk - dv)
    t["q"], t["beta"], t["state_init"] = t["k"], torch.ones_like(t["beta"]), 2000.0 * t["state_init"]
    check(t)
