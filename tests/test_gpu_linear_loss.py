"""The cross entropy of a projection to a vocabulary against float64.

Tolerances.  A logit is a sum of D products, exact for bf16 inputs and off by 3 2^-24
of their size for fp32 ones (three bf16 parts an operand), added in fp32: off by at most
d = (D + 8) 2^-24 max_v sum |h w| (and another 2^-22 |logit| where logits are as large as
16, for exp2's argument).  A loss is off by 2 d and the roundings of the sums of
exponentials over up to 64 elements, their joins and the logarithm: 80 2^-24 of a factor,
so 5e-6.  A probability less its target's one is off by 2 d + 5e-6 of the probability, and,
for bf16 inputs, rounded to bf16: 2^-8 of the value (up to 64 tokens: the sum of 2 parts,
2^-16), the sum of 3 parts for fp32: 3 2^-24.
The gradients add up terms P W and P H: (V + 16) 2^-24, (N + 16) 2^-24 of the sum of their
sizes, and bf16 results half a unit in the last place, 2^-8.
"""
import pytest
import torch

from orthossm_amd import linear_cross_entropy, linear_cross_entropy_backward, linear_cross_entropy_forward

pytestmark = pytest.mark.gpu
IGNORE = -100


def make(N, D, V, dtype=torch.float32, seed=0, ignored=0.0):
    gen = torch.Generator().manual_seed(seed)
    weight = (2.0 * torch.randn(V, D, generator=gen) / D ** 0.5).to(dtype)
    targets = torch.randint(V, (N,), generator=gen)
    hidden = (torch.randn(N, D, generator=gen) + 0.5 * weight[targets].float()).to(dtype)
    if ignored:
        targets[torch.rand(N, generator=gen) < ignored] = IGNORE
    return hidden, weight, targets


def check(dev, hidden, weight, targets, ignore=IGNORE):
    N, D, V = *hidden.shape, weight.shape[0]
    bf = hidden.dtype == torch.bfloat16
    h, w = hidden.double(), weight.double()
    keep = (targets != ignore).nonzero()[:, 0]
    t = targets[keep].long()
    # (a row that does not count may hold anything)
    h = torch.zeros_like(h).index_copy(0, keep, h[keep])
    z = h[keep] @ w.t()
    lse = torch.logsumexp(z, -1)
    at = torch.arange(keep.numel())
    each = lse - z[at, t]
    size = (h[keep].abs() @ w.abs().t()).max(-1, keepdim=True).values if keep.numel() else torch.zeros(0, 1, dtype=torch.float64)
    d = 2.0 ** -24 * (D + 8) * size + 2.0 ** -22 * z.abs().max(-1, keepdim=True).values.clamp(min=16)
    hd, wd, td = (x.to(dev) for x in (hidden, weight, targets))
    losses, got_lse = (x.double().cpu() for x in linear_cross_entropy_forward(hd, wd, td, ignore_index=ignore))
    bound = 2 * d[:, 0] + 5e-6
    assert ((losses[keep] - each).abs() <= bound).all() and ((got_lse[keep] - lse).abs() <= bound + 2.0 ** -23 * lse.abs()).all()
    gone = targets == ignore
    assert (losses[gone] == 0).all() and (got_lse[gone] == 0).all()
    g = torch.rand(N, generator=torch.Generator().manual_seed(1)) + 0.5
    P = torch.softmax(z, -1)
    off = P * (2 * d + 5e-6)
    P[at, t] -= 1.0
    # rounded to bf16, once and (with each token's own gradient in it) as it is used
    off = off + P.abs() * ((2.0 ** -16 if N <= 64 else 2.0 ** -8) if bf else 4 * 2.0 ** -24)
    leaves = [hd.requires_grad_(), wd.requires_grad_()]
    for reduction, each_g in (("none", g[keep].double()), ("sum", torch.full((keep.numel(),), 0.75, dtype=torch.float64)),
                              ("mean", torch.full((keep.numel(),), 0.75 / max(1, keep.numel()), dtype=torch.float64))):
        loss = linear_cross_entropy(*leaves, td, ignore_index=ignore, reduction=reduction)
        assert loss.dtype == torch.float32
        want = each if reduction == "none" else each.sum() if reduction == "sum" else each.sum() / max(1, keep.numel())
        tol = bound if reduction == "none" else bound.sum() + 2.0 ** -23 * want if reduction == "sum" else \
            (bound.sum() / max(1, keep.numel()) + 2.0 ** -22 * want)
        got = loss.detach().double().cpu()
        assert ((got[keep] if reduction == "none" else got) - want).abs().le(tol).all(), reduction
        gh, gw = torch.autograd.grad(loss, leaves, g.to(dev) if reduction == "none" else torch.tensor(0.75, device=dev))
        assert gh.dtype == hidden.dtype and gw.dtype == weight.dtype
        Pg, offg = P * each_g[:, None], off * each_g[:, None]
        half = 2.0 ** -8 if bf else 0.0
        dh = torch.zeros_like(h).index_copy(0, keep, Pg @ w)
        th = torch.zeros_like(h).index_copy(0, keep, (offg + 2.0 ** -24 * (V + 16) * Pg.abs()) @ w.abs())
        over = (gh.double().cpu() - dh).abs() - th - half * (dh.abs() + th) - 1e-30
        assert over.max().item() <= 0, (reduction, "grad_hidden", over.max().item())
        dw = Pg.t() @ h[keep]
        tw = (offg + 2.0 ** -24 * (keep.numel() + 16) * Pg.abs()).t() @ h[keep].abs()
        over = (gw.double().cpu() - dw).abs() - tw - half * (dw.abs() + tw) - 1e-30
        assert over.max().item() <= 0, (reduction, "grad_weight", over.max().item())
        assert (gh[gone.to(dev)] == 0).all()


TYPES = [torch.float32, torch.bfloat16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N", [1, 2, 63, 64, 65, 127, 129, 255, 257, 700])
def test_tokens(dev, N, dtype):
    check(dev, *make(N, 96, 300, dtype, seed=N))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [1, 2, 3, 127, 128, 129, 255, 257, 1000, 1025])
def test_vocabularies(dev, V, dtype):
    check(dev, *make(70, 64, V, dtype, seed=V))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [1, 3, 8, 31, 63, 64, 65, 100, 128, 200, 256, 257, 512, 1000])
def test_widths(dev, D, dtype):
    check(dev, *make(40, D, 150, dtype, seed=D))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N", [1, 64, 65, 129])
def test_few_tokens_over_many_classes(dev, N, dtype):
    check(dev, *make(N, 64, 49400, dtype, seed=N, ignored=0.2 if N > 1 else 0.0))
    check(dev, *make(N, 2100, 700, dtype, seed=N))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ignored", [0.02, 0.5, 0.95, 1.1])
def test_ignored_tokens_may_hold_anything(dev, ignored, dtype):
    for N, D in ((300, 80), (300, 64), (600, 64)):
        hidden, weight, targets = make(N, D, 400, dtype, seed=1, ignored=ignored)
        hidden[targets == IGNORE] = float("nan")
        check(dev, hidden, weight, targets)


# The three tile sizes of each product, several pieces of the vocabulary.
@pytest.mark.parametrize("dtype,N,D,V", [(torch.bfloat16, 4000, 64, 4000), (torch.bfloat16, 2100, 130, 2600),
                                         (torch.float32, 1500, 64, 3000), (torch.float32, 4100, 33, 4100),
                                         (torch.bfloat16, 70000, 64, 3000), (torch.float32, 40000, 16, 1500),
                                         (torch.bfloat16, 300, 1024, 9000), (torch.bfloat16, 5, 64, 70001)])
def test_sizes(dev, dtype, N, D, V):
    check(dev, *make(N, D, V, dtype, seed=2, ignored=0.1))


def test_another_index_is_ignored(dev):
    hidden, weight, targets = make(50, 32, 60, seed=3)
    targets[::3] = 7
    check(dev, hidden, weight, targets, ignore=7)


@pytest.mark.parametrize("dtype", TYPES)
def test_targets_outside(dev, dtype):
    """NaN, where the token has a part; nothing is read or written outside."""
    hidden, weight, targets = (t.to(dev) for t in make(30, 32, 40, dtype, seed=4))
    targets[3], targets[5], targets[6] = 40, -1, 2 ** 40
    losses, lse = linear_cross_entropy_forward(hidden, weight, targets)
    bad = torch.zeros(30, dtype=torch.bool, device=dev)
    bad[[3, 5, 6]] = True
    assert torch.isnan(losses[bad]).all() and torch.isfinite(losses[~bad]).all()
    gh, gw = linear_cross_entropy_backward(torch.ones_like(losses), hidden, weight, targets, lse)
    assert torch.isnan(gh[bad]).all() and torch.isfinite(gh[~bad]).all() and torch.isnan(gw).all()
    assert torch.isnan(linear_cross_entropy(hidden, weight, targets))


def test_large_and_infinite_logits(dev):
    hidden, weight, targets = make(20, 16, 30, seed=5)
    check(dev, 40 * hidden, weight, targets)
    check(dev, hidden, torch.zeros_like(weight), targets)
    hidden, weight = hidden.abs() + 0.1, weight.clone()
    weight[4] = -float("inf")          # a class that no token can have
    targets[targets == 4] = 5
    losses, _ = linear_cross_entropy_forward(hidden.to(dev), weight.to(dev), targets.to(dev))
    rest = [v for v in range(30) if v != 4]
    z = hidden.double() @ weight[rest].double().t()
    at = torch.tensor([rest.index(int(t)) for t in targets])
    want = torch.logsumexp(z, -1) - z[torch.arange(20), at]
    # (an infinite fp32 weight has no three parts: NaN.  In bf16 it is one)
    half = linear_cross_entropy_forward(hidden.bfloat16().to(dev), weight.bfloat16().to(dev), targets.to(dev))[0]
    z = hidden.bfloat16().double() @ weight[rest].bfloat16().double().t()
    want = torch.logsumexp(z, -1) - z[torch.arange(20), at]
    assert ((half.double().cpu() - want).abs() <= 1e-4).all()
    assert torch.isnan(losses).all() or ((losses.double().cpu() - want).abs() <= 1e-1).all()


def test_confident_tokens(dev):
    """A loss far below its logits' size keeps its own digits."""
    weight = torch.eye(16)
    hidden = 30.0 * torch.eye(16)
    losses, _ = linear_cross_entropy_forward(hidden.to(dev), weight.to(dev), torch.arange(16, device=dev))
    want = torch.log1p(15 * torch.exp(torch.tensor(-30.0, dtype=torch.float64)))
    assert (losses.double().cpu() - want).abs().max() <= 2.0 ** -24


def test_layouts_and_types(dev):
    hidden, weight, targets = (t.to(dev) for t in make(60, 64, 100, torch.bfloat16, seed=6))
    want = linear_cross_entropy_forward(hidden, weight, targets)
    wide_h, wide_w = torch.zeros(60, 71, dtype=hidden.dtype, device=dev), torch.zeros(100, 72, dtype=hidden.dtype, device=dev)
    wide_h[:, 3:67], wide_w[:, 8:] = hidden, weight
    odd = torch.zeros(100, 67, dtype=hidden.dtype, device=dev)
    odd[:, 1:65] = weight
    for h, w in ((wide_h[:, 3:67], weight), (hidden, wide_w[:, 8:]), (hidden, odd[:, 1:65]),
                 (hidden.t().contiguous().t(), weight.t().contiguous().t())):
        assert all(torch.equal(p, q) for p, q in zip(linear_cross_entropy_forward(h, w, targets), want))
    for t in (targets.int(), targets.short(), torch.stack([targets, targets], -1)[:, 0]):
        assert torch.equal(linear_cross_entropy_forward(hidden, weight, t)[0], want[0])
    shaped = linear_cross_entropy(hidden.view(5, 12, 64), weight, targets.view(5, 12), reduction="none")
    assert shaped.shape == (5, 12) and torch.equal(shaped.flatten(), want[0])
    one = hidden[:1].expand(60, 64)      # strides of zero
    assert torch.equal(linear_cross_entropy_forward(one, weight, targets)[0], linear_cross_entropy_forward(one.contiguous(), weight, targets)[0])
    g = torch.rand(60, device=dev)
    grads = linear_cross_entropy_backward(g, hidden, weight, targets, want[1])
    again = linear_cross_entropy_backward(torch.stack([g, g], -1)[:, 0], wide_h[:, 3:67], wide_w[:, 8:], targets, want[1])
    assert all(torch.equal(p, q) for p, q in zip(grads, again))
    h16, w32 = hidden.half().requires_grad_(), weight.float().requires_grad_()
    gh, gw = torch.autograd.grad(linear_cross_entropy(h16, w32, targets), (h16, w32))
    assert gh.dtype == torch.float16 and gw.dtype == torch.float32


def test_needs(dev):
    hidden, weight, targets = (t.to(dev) for t in make(90, 48, 200, torch.bfloat16, seed=7))
    _, lse = linear_cross_entropy_forward(hidden, weight, targets)
    g = torch.rand(90, device=dev)
    whole = linear_cross_entropy_backward(g, hidden, weight, targets, lse)
    only_h = linear_cross_entropy_backward(g, hidden, weight, targets, lse, need_weight=False)
    only_w = linear_cross_entropy_backward(g, hidden, weight, targets, lse, need_hidden=False)
    assert torch.equal(only_h[0], whole[0]) and only_h[1] is None and torch.equal(only_w[1], whole[1]) and only_w[0] is None
    for i in range(2):
        mine = [t.clone().requires_grad_(j == i) for j, t in enumerate((hidden, weight))]
        linear_cross_entropy(*mine, targets).backward()
        assert [t.grad is not None for t in mine] == [j == i for j in range(2)]


def test_gradients_against_differences(dev):
    """Central differences of the kernel's forward, h = 2^-5."""
    hidden, weight, targets = (t.to(dev) for t in make(60, 24, 50, seed=8, ignored=0.2))
    leaves = [hidden.requires_grad_(), weight.requires_grad_()]
    grads = torch.autograd.grad(linear_cross_entropy(*leaves, targets, reduction="sum"), leaves)
    h, gen = 2.0 ** -5, torch.Generator().manual_seed(0)
    for i, grad in enumerate(grads):
        way = torch.randn(grad.shape, generator=gen).to(dev)
        way /= way.norm()
        up, down = (linear_cross_entropy_forward(*(t.detach() + s * h * way if j == i else t.detach() for j, t in enumerate(leaves)),
                                                 targets)[0].double().sum() for s in (1.0, -1.0))
        got = (grad.double() * way.double()).sum().item()
        assert abs((up - down).item() / (2 * h) - got) <= 4 * h * h * grad.norm().item() + 1e-3


def test_empty(dev):
    weight = torch.ones(7, 5, device=dev, requires_grad=True)
    hidden = torch.zeros(0, 5, device=dev, requires_grad=True)
    targets = torch.zeros(0, dtype=torch.int64, device=dev)
    for reduction in ("mean", "sum", "none"):
        loss = linear_cross_entropy(hidden, weight, targets, reduction=reduction)
        gh, gw = torch.autograd.grad(loss, (hidden, weight), torch.ones_like(loss))
        assert gh.shape == (0, 5) and (gw == 0).all() and (loss == 0).all()
    w16 = torch.ones(3, 5, dtype=torch.bfloat16, device=dev)
    gw = linear_cross_entropy_backward(torch.zeros(0, device=dev), hidden.detach().bfloat16(), w16, targets, torch.zeros(0, device=dev))[1]
    assert (gw == 0).all()


def test_same_bits_on_every_run_and_graph(dev):
    hidden, weight, targets = (t.to(dev) for t in make(1500, 192, 5000, torch.bfloat16, seed=9, ignored=0.2))
    g = torch.rand(1500, device=dev)

    def everything():
        losses, lse = linear_cross_entropy_forward(hidden, weight, targets)
        return (losses, lse, *linear_cross_entropy_backward(g, hidden, weight, targets, lse))

    want = everything()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = everything()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for p, q, r in zip(want, everything(), held):
            assert torch.equal(p, q) and torch.equal(p, r)


def test_two_streams_at_once(dev):
    ins = [[t.to(dev) for t in make(900, 128, 3000, torch.bfloat16, seed=s)] for s in (10, 11)]
    want = [linear_cross_entropy_forward(*i) for i in ins]
    streams = [torch.cuda.Stream(dev) for _ in ins]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for i, s in zip(ins, streams):
            with torch.cuda.stream(s):
                got.append(linear_cross_entropy_forward(*i))
    torch.cuda.synchronize()
    for k, g in enumerate(got):
        assert all(torch.equal(p, q) for p, q in zip(g, want[k % 2]))


def test_refusals(dev):
    h, w, t = torch.zeros(4, 8, device=dev), torch.zeros(5, 8, device=dev), torch.zeros(4, dtype=torch.int64, device=dev)
    for bad in (lambda: linear_cross_entropy(h, w[:, :7], t), lambda: linear_cross_entropy(h, w[0], t), lambda: linear_cross_entropy(h, None, t),
                lambda: linear_cross_entropy(h, w, t[:3]), lambda: linear_cross_entropy(h, w, t.float()), lambda: linear_cross_entropy(h, w, t.bool()),
                lambda: linear_cross_entropy(h, w, t.cpu()), lambda: linear_cross_entropy(h, w.cpu(), t), lambda: linear_cross_entropy(h, w[:0], t),
                lambda: linear_cross_entropy([1.0], w, t), lambda: linear_cross_entropy(h, w, t, reduction="max"),
                lambda: linear_cross_entropy_backward(torch.ones(3, device=dev), h, w, t, torch.zeros(4, device=dev)),
                lambda: linear_cross_entropy_backward(torch.ones(4, device=dev), h, w, t, torch.zeros(3, device=dev))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="ROCm GPU only"):
        linear_cross_entropy(h.cpu(), w.cpu(), t.cpu())
