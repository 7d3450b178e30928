"""The cross entropy of a projection to a vocabulary in forms of their own, by the
bounds of test_gpu_linear_loss."""
import pytest
import torch
from test_gpu_linear_loss import check, make

from orthossm_amd import linear_cross_entropy_backward, linear_cross_entropy_forward

pytestmark = pytest.mark.gpu


# Several pieces of copied weights: 23808 classes of 2112 in three parts, 36096 of 4160 in one.
@pytest.mark.parametrize("dtype,N,D,V", [(torch.float32, 5, 2100, 25000), (torch.float32, 300, 2100, 24001),
                                         (torch.bfloat16, 3, 4100, 37000), (torch.bfloat16, 70, 4100, 36200)])
def test_few_tokens_over_pieces_of_copied_weights(dev, dtype, N, D, V):
    check(dev, *make(N, D, V, dtype, seed=N, ignored=0.2 if N > 5 else 0.0))


def summed(hidden, weight):
    """Logits in float64, a product with an infinity an infinity."""
    return (hidden.double()[:, None] * weight.double()[None]).sum(-1)


@pytest.mark.parametrize("N,D,V", [(20, 16, 30), (150, 100, 700), (700, 65, 300)])
@pytest.mark.parametrize("whole", [False, True])
def test_infinite_fp32_weights_leave_a_class_out(dev, N, D, V, whole):
    """Against the definition in 64 bits: P and the loss of what is left, the class's own
    gradient 0; 0 times infinity, NaN, in grad_hidden's columns where there is one."""
    hidden, weight, targets = make(N, D, V, seed=N)
    hidden[:, 0] = hidden[:, 0].abs() + 0.1
    out = [1, 4, V - 1]
    for v in out:
        targets[targets == v] = 5
    if whole:
        hidden = hidden.abs() + 0.1
        weight[out] = -float("inf")
    else:
        weight[out, 0] = -float("inf")
    z = summed(hidden, weight)
    assert (z[:, out] == -float("inf")).all()
    at = torch.arange(N)
    lse = torch.logsumexp(z, -1)
    each = lse - z[at, targets]
    left = [v for v in range(V) if v not in out]
    # (the bounds of test_gpu_linear_loss)
    size = (hidden.double().abs() @ weight[left].double().abs().t()).max(-1).values
    d = 2.0 ** -24 * (D + 8) * size + 2.0 ** -22 * z[:, left].abs().max(-1).values.clamp(min=16)
    hd, wd, td = (t.to(dev) for t in (hidden, weight, targets))
    losses, got_lse = linear_cross_entropy_forward(hd, wd, td)
    bound = 2 * d + 5e-6
    assert ((losses.double().cpu() - each).abs() <= bound).all()
    assert ((got_lse.double().cpu() - lse).abs() <= bound + 2.0 ** -23 * lse.abs()).all()
    gh, gw = (t.double().cpu() for t in linear_cross_entropy_backward(torch.ones_like(losses), hd, wd, td, got_lse))
    P = torch.softmax(z, -1)
    off = P * (2 * d[:, None] + 5e-6)
    P[at, targets] -= 1.0
    off = off + 4 * 2.0 ** -24 * P.abs()
    dw = P.t() @ hidden.double()
    tol = (off + 2.0 ** -24 * (N + 16) * P.abs()).t() @ hidden.double().abs()
    assert ((gw - dw).abs() <= tol + 1e-30).all() and (gw[out] == 0).all()
    assert torch.isnan(gh).all() if whole else torch.isnan(gh[:, 0]).all()
    if not whole:
        dh = P[:, left] @ weight[left, 1:].double()
        tol = (off + 2.0 ** -24 * (V + 16) * P.abs())[:, left] @ weight[left, 1:].double().abs()
        assert ((gh[:, 1:] - dh).abs() <= tol + 1e-30).all()


def test_a_target_that_is_left_out_has_an_infinite_loss(dev):
    hidden, weight, targets = make(20, 16, 30, seed=5)
    hidden = hidden.abs() + 0.1
    weight[4] = -float("inf")
    targets[:] = 3
    targets[7] = 4
    for dtype in (torch.float32, torch.bfloat16):
        losses, lse = linear_cross_entropy_forward(hidden.to(dev, dtype), weight.to(dev, dtype), targets.to(dev))
        assert losses[7] == float("inf") and torch.isfinite(lse).all() and torch.isfinite(losses).sum() == 19


@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_the_largest_fp32_values_have_three_parts(dev, sign):
    """What bf16 would round to infinity: 3.4e38 times 2^-125 in a logit of 8."""
    hidden, weight, targets = make(40, 33, 50, seed=6)
    hidden[:, 0] = 2.0 ** -125
    weight[:, 0] = 0.0
    weight[::7, 0] = sign * 3.4e38
    z = summed(hidden, weight)
    size = (hidden.double().abs()[:, None] * weight.double().abs()[None]).sum(-1).max(-1).values
    bound = 2 * (2.0 ** -24 * (33 + 8) * size + 2.0 ** -22 * z.abs().max(-1).values.clamp(min=16)) + 5e-6
    losses = linear_cross_entropy_forward(*(t.to(dev) for t in (hidden, weight, targets)))[0].double().cpu()
    assert ((losses - (torch.logsumexp(z, -1) - z[torch.arange(40), targets])).abs() <= bound).all()


def test_infinite_hidden_values_make_nan_of_their_own_tokens_only(dev):
    hidden, weight, targets = make(80, 32, 60, seed=7)
    for dtype in (torch.float32, torch.bfloat16):
        h = hidden.clone()
        h[[3, 70], 5] = float("inf")
        losses, _ = linear_cross_entropy_forward(h.to(dev, dtype), weight.to(dev, dtype), targets.to(dev))
        clean, _ = linear_cross_entropy_forward(hidden.to(dev, dtype), weight.to(dev, dtype), targets.to(dev))
        assert torch.isnan(losses[[3, 70]]).all()
        rest = [n for n in range(80) if n not in (3, 70)]
        assert torch.equal(losses[rest], clean[rest])
