"""GatedDeltaLayer and the example that trains and serves with it."""
import importlib.util
import os

import pytest
import torch
import torch.nn.functional as F

from oracle import delta as O
from orthossm_amd import GatedDeltaLayer

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_constructor_refuses_odd_heads():
    with pytest.raises(ValueError, match="multiple"):
        GatedDeltaLayer(64, 4, n_qk_heads=3)


def _reference(m, x, state=None):
    """The layer in float64 on the CPU, from the same parameters."""
    p = {n: t.detach().double().cpu() for n, t in m.named_parameters()}
    x = x.double().cpu()
    B, S, D = x.shape
    h = F.layer_norm(x, (D,), p["norm_weight"], p["norm_bias"], m.eps)
    q, k, v, a, b = (h @ p["in_proj.weight"].T).split(m.splits, -1)
    q, k = (F.normalize(t.reshape(B, S, m.n_qk_heads, m.head_dim), dim=-1) for t in (q, k))
    g = -torch.exp(p["a_log"]) * F.softplus(a + p["a_bias"])
    out, fin = O.gated_delta(q, k, v.reshape(B, S, m.n_heads, m.value_dim), g, torch.sigmoid(b),
                             state_init=None if state is None else state.double().cpu())
    return x + out.flatten(2) @ p["out_proj.weight"].T, fin


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(), dict(n_heads=4, n_qk_heads=2, head_dim=24, value_dim=40)])
def test_layer_forward_and_step(dev, kw):
    """fp32 tolerance: torch's projections (sums of 96 terms, 96^(1/2) 2^-24 =
    6e-7, twice) on top of the operators' 8e-6 each: 2e-5."""
    torch.manual_seed(0)
    m = GatedDeltaLayer(96, **kw).to(dev)
    x = torch.randn(2, 90, 96, device=dev)
    with torch.no_grad():
        y, state = m(x)
        want, fin = _reference(m, x)
        assert (y.double().cpu() - want).norm() <= 2e-5 * want.norm()
        assert (state.double().cpu() - fin).norm() <= 2e-5 * fin.norm()
        # a prompt, then token by token at slots of a pool
        lengths = torch.tensor([80, 86], device=dev)
        y0, state = m(x, lengths=lengths)
        assert torch.equal(y0[0, 80:], x[0, 80:])
        pool, slots = m.new_state(5), torch.tensor([3, 1], device=dev)
        pool[slots] = state
        for t in range(4):
            out = m.step(x[torch.arange(2), lengths + t], pool, slots)
            for b in range(2):
                ref = want[b, int(lengths[b]) + t]
                assert (out[b].double().cpu() - ref).norm() <= 2e-5 * ref.norm()


@pytest.mark.gpu
def test_layer_gradients(dev):
    torch.manual_seed(1)
    m = GatedDeltaLayer(64, 4).to(dev)
    x = torch.randn(2, 70, 64, device=dev)
    way = torch.randn(2, 70, 64, device=dev)
    (m(x)[0] * way).sum().backward()
    p = dict(m.named_parameters())
    h = 2.0 ** -7
    gen = torch.Generator().manual_seed(2)
    for name, t in p.items():      # differences along a random direction, as in the operators' tests
        d = torch.randn(t.shape, generator=gen).to(dev)
        d /= d.norm()
        with torch.no_grad():
            vals = []
            for s in (1.0, -1.0):
                t.add_(s * h * d)
                vals.append((m(x)[0].double() * way.double()).sum().item())
                t.sub_(s * h * d)
        want = (vals[0] - vals[1]) / (2 * h)
        got = (t.grad.double() * d.double()).sum().item()
        assert abs(got - want) <= 4 * h * h * t.grad.norm().item() + 2e-3, name


@pytest.mark.gpu
def test_example_learns_and_serves(dev):
    spec = importlib.util.spec_from_file_location("delta_training", os.path.join(ROOT, "examples", "delta_training.py"))
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    torch.manual_seed(0)
    gen = torch.Generator().manual_seed(0)
    model = ex.RecallModel(64, 2).to(dev)
    losses, norms = ex.train(model, 60, gen)
    assert torch.isfinite(losses).all() and (norms > 0).all()
    assert losses[-10:].mean() < losses[:10].mean()
    share, worst = ex.serve(model, gen, rows=16)
    assert 0.0 <= share <= 1.0 and worst <= 1e-3


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float64])
def test_states_are_fp32_whatever_the_default_type(dtype):
    m = GatedDeltaLayer(32, 2)
    torch.set_default_dtype(dtype)
    try:
        assert m.new_state(3).dtype == torch.float32
    finally:
        torch.set_default_dtype(torch.float32)
