"""bf16 results of the gated delta rule against the float64 ones, rounded to bf16.

A bound on the distance to the exact value has to allow the rounding itself,
2^-8 of an element, and hides arithmetic a hundred times too coarse.  The
distance to the exact value rounded to bf16 does not: it is zero but where a
rounding goes the other way.  For a result off by e that happens to an element
with probability |e| / ulp and costs an ulp, ulp <= 2^-7 |y|, so the expected
square of the distance is at most 2^-7 sum |y| |e| <= 2^-7 |y| |e|, and with
|e| <= 8e-6 |y|, the bound that fp32 results are held to (test_gpu_delta.py),
the distance is 2.5e-4 |y|.  The tensors have 50000 elements and more, so that
the share of turned roundings is near what is expected.
"""
import pytest
import torch

from oracle import delta as O
from orthossm_amd import gated_delta
from test_gpu_delta import FP32, args, make, on

TURNED = (2.0 ** -7 * FP32) ** 0.5


def distance(got, want):
    want = want.double()
    return ((got.double().cpu() - want.bfloat16().double()).norm() / want.norm()).item()


def test_the_measure_sees_one_bf16_part():
    """Products whose operands are rounded to bf16 first, of fp32 sums."""
    gen = torch.Generator().manual_seed(0)
    a, b = (torch.randn(400, 64, generator=gen, dtype=torch.float64) for _ in range(2))
    want = a @ b.T
    assert distance((a.float() @ b.float().T).bfloat16(), want) <= TURNED
    assert distance((a.bfloat16().float() @ b.float().T).bfloat16(), want) > 4 * TURNED


@pytest.mark.gpu
@pytest.mark.parametrize("same_keys", [False, True])
@pytest.mark.parametrize("B,S,H,Hk,dk,dv", [(2, 150, 4, 4, 64, 64), (4, 150, 4, 2, 50, 80), (1, 140, 4, 4, 128, 128),
                                            (2, 140, 4, 4, 96, 48)])
def test_against_rounded_results(dev, B, S, H, Hk, dk, dv, same_keys):
    """Also with equal keys and a start state a thousand times the values,
    where what is read of it and what the updates add nearly cancel."""
    t = make(B, S, H, dk, dv, Hk, torch.bfloat16, seed=S + dk, same_keys=same_keys)
    if same_keys:
        t["q"], t["state_init"] = t["k"], 2000.0 * t["state_init"]
    want = O.gated_delta_grads(*args(t), t["grad_out"], t["grad_state"], state_init=t["state_init"])
    d = on(t, dev)
    leaves = [x.requires_grad_() for x in (*args(d), d["state_init"])]
    out, fin = gated_delta(*leaves[:5], state_init=leaves[5], return_state=True)
    grads = torch.autograd.grad((out, fin), leaves, (d["grad_out"], d["grad_state"]))
    for name, got, ref in (("out", out.detach(), want[0]), *zip(("grad_q", "grad_k", "grad_v"), grads, want[2:5])):
        assert got.dtype == torch.bfloat16
        assert distance(got, ref) <= TURNED, name
