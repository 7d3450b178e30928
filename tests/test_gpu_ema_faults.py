"""Waits of the gated EMA's tiles that give up, forced from the host: they leave
NaN and the fault word.  Tiles by index (8 lane-blocks) and drawn (6)."""
import numpy as np
import pytest
import torch
from test_gpu_gated_ema import make

from orthossm_amd import _native as nat
from orthossm_amd import ema, gated_ema, gated_ema_backward, gated_ema_forward, ops

pytestmark = pytest.mark.gpu
SHAPES = [(8, 128), (3, 256)]


def nan_or_equal(got, want, what):
    """Every element of `got` is NaN or bit-equal to `want`; whether one is NaN."""
    g, w = (t.detach().float().cpu().numpy() for t in (got, want))
    nan = np.isnan(g)
    assert not np.isnan(w).any() and np.array_equal(g[~nan].view(np.uint32), w[~nan].view(np.uint32)), what
    return bool(nan.any())


def until_one_gives_up(run):
    """Whether a wait gives up depends on timing: up to four runs."""
    for _ in range(4):
        old = ops.set_poll_limit_zero(True)
        try:
            if run():
                return
        finally:
            ops.set_poll_limit_zero(old)
    pytest.fail("no wait gave up")


@pytest.mark.parametrize("B,D", SHAPES)
def test_waits_that_give_up_leave_nan(dev, B, D, monkeypatch):
    """A word that is not there at its first read gives up at once: every block
    ends, what depends on the lost value is NaN, the rest as ever, and so is the next
    call."""
    x, gate, init, go, gs = (t.to(dev) for t in make(B, 20000, D, seed=1))

    def forward():
        return gated_ema_forward(x, gate, state_init=init, return_state=True)

    monkeypatch.setattr(ema, "_fast", lambda: None)     # (a graph whose backward takes the aid)
    leaves = [t.requires_grad_() for t in (x, gate, init)]
    outs = gated_ema(*leaves[:2], state_init=leaves[2], return_state=True)

    def backward():
        return torch.autograd.grad(outs, leaves, (go, gs), retain_graph=True)

    for run in (forward, backward):
        want = [t.detach().clone() for t in run()]
        until_one_gives_up(lambda: any([nan_or_equal(g, w, run.__name__) for g, w in zip(run(), want)]))
        assert all(torch.equal(g, w) for g, w in zip(run(), want))


@pytest.mark.parametrize("B,D", SHAPES)
def test_waits_that_give_up_raise_where_faults_are_checked(dev, B, D):
    x, gate, init, go, gs = (t.to(dev) for t in make(B, 20000, D, seed=2))
    runs = [lambda: gated_ema_forward(x, gate, state_init=init),
            lambda: gated_ema_backward(x, gate, go, state_init=init, grad_state=gs, need_init=True)]
    old = ops.set_fault_check(True)
    try:
        for run in runs:
            def gives_up():
                try:
                    run()
                except nat.OsmError as e:
                    assert "gated_ema" in str(e) and "look-back wait gave up" in str(e) and "OSM_E_FAULT" in str(e)
                    return True
            run()                      # (nothing to report)
            until_one_gives_up(gives_up)
            run()
    finally:
        ops.set_fault_check(old)
