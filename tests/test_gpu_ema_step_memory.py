"""Tokens of the gated EMA's step that lie in the memory of the states."""
import pytest
import torch
from test_gpu_ema_block_loss_paths import path, through_ctypes  # noqa: F401

from orthossm_amd import gated_ema_step

pytestmark = pytest.mark.gpu
B, D = 4, 24


def rand(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda()


def want(x, gate, state):
    a, o = torch.sigmoid(gate.double()), torch.sigmoid(-gate.double())
    return a * state.double() + o * x.double()


def near(got, ref):
    # (the sigmoids, two products and a sum: a few units of 2^-24 of values up to 4)
    assert (got.double() - ref).abs().max().item() <= 2.0 ** -20


def test_tokens_in_other_rows_states_are_refused(dev, path):  # noqa: F811
    pool, other = rand(6, D, seed=1), rand(B, D, seed=2)
    before = pool.clone()
    slots = torch.tensor([2, 0, 3, 1], device=dev)
    half = pool.view(torch.bfloat16)
    for x, gate, s in ((pool[:B], other, slots), (other, pool[:B], slots), (pool[1:5], other, None), (other, pool[2:], None),
                       (pool[:1].expand(B, D), other, None), (pool[:B].flatten()[3:-1].as_strided((B, D), (D - 1, 1)), other, None),
                       (half[:B, :D], other.bfloat16(), None)):
        with pytest.raises(ValueError, match="shares memory with state"):
            gated_ema_step(x, gate, pool, slots=s)
        assert torch.equal(pool, before)


def test_tokens_beside_the_states_or_the_states_themselves(dev, path):  # noqa: F811
    gate, wide = rand(B, D, seed=3), rand(B, 3 * D, seed=4)
    for slots in (None, torch.tensor([2, 0, 3, 1], device=dev)):
        for x, state in ((wide[:, :D], wide[:, D:2 * D]), (wide[:, 2 * D:], wide[:, :D]), (wide[:, :D], wide[:, 2 * D:]),
                         (wide[:1, :D].expand(B, D), wide[:, D:2 * D]), (wide[::2, :D][[0, 1, 1, 0]], wide[:, D:2 * D])):
            at = torch.arange(B, device=dev) if slots is None else slots
            ref = want(x, gate, state[at])
            near(gated_ema_step(x, gate, state, slots=slots), ref)
            near(state[at], ref)
    state = rand(B + 2, D, seed=5)
    rest, ref = state[B:].clone(), want(state[:B], gate, state[:B])
    near(gated_ema_step(state[:B], gate, state), ref)
    near(state[:B], ref)
    assert torch.equal(state[B:], rest)
    ref = want(gate, state[:B], state[:B])
    near(gated_ema_step(gate, state[:B], state), ref)
    near(state[:B], ref)


def test_many_steps_in_one_pool(dev, path):  # noqa: F811
    """Layers whose states share a tensor, the one's output the next one's input."""
    pool, gate = rand(3 * B, D, seed=6), rand(B, D, seed=7)
    x, ref = rand(B, D, seed=8), None
    for layer in range(3):
        state = pool[layer * B:(layer + 1) * B]
        ref = want(x, gate, state)
        x = gated_ema_step(x, gate, state)
        near(x, ref)
        near(state, ref)
