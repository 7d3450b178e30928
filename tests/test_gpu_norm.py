"""Layer norm against float64.

Tolerances.  A row's sums add at most 16 elements a thread, then a tree of ten
levels: 26 roundings of 2^-24 relative to the row's absolute mean, which is at
most five standard deviations here, so 8e-6 of a result's size.  bf16 results
add half a unit in the last place, 2^-8 of each element.  dw and db add up to
200 terms in a row (a thread's rows, four row groups, an eighth of the lines of
sums): 200 2^-24 of the sum of the terms' sizes.  dx is a difference (for one
or two elements a row nearly all of it cancels), so its bound is relative to
the size of its terms too.
"""
import pytest
import torch

from orthossm_amd import layer_norm, layer_norm_backward, layer_norm_forward

FP32 = 8e-6
BF16 = 2.0 ** -8 + FP32
SUMS = 200 * 2.0 ** -24


def make(shape, dtype=torch.float32, seed=0):
    gen = torch.Generator().manual_seed(seed)
    D = shape[-1]

    def rand(*s):
        return torch.randn(*s, generator=gen)

    x = (rand(*shape) * (1 + rand(*shape[:-1], 1).abs()) + rand(*shape[:-1], 1)).to(dtype)
    return x, 1 + 0.3 * rand(D), 0.3 * rand(D), rand(*shape).to(dtype)


def reference(x, w, b, dy, eps):
    """y, dx, dw, db and the sums of the sizes of the gradients' terms."""
    x, dy = x.double(), dy.double()
    w = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else w.double()
    mean, var = x.mean(-1, keepdim=True), x.var(-1, correction=0, keepdim=True)
    rstd = (var + eps) ** -0.5
    xh = (x - mean) * rstd
    y = xh * w + (0 if b is None else b.double())
    g = dy * w
    dx = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    tx = rstd * (g.abs() + g.abs().mean(-1, keepdim=True) + xh.abs() * (g * xh).abs().mean(-1, keepdim=True))
    lead = tuple(range(x.dim() - 1))
    terms = dy * xh
    return y, dx, terms.sum(lead), dy.sum(lead), tx, terms.abs().sum(lead), dy.abs().sum(lead)


def close(got, want, tol, what, terms=None):
    got = got.double().cpu()
    assert got.shape == want.shape and torch.isfinite(got).all(), what
    err, size = (got - want).norm().item(), (want if terms is None else terms).norm().item()
    assert err <= tol * size + 1e-12, f"{what}: {err / (size + 1e-300):.2e} of the norm, {tol:.1e} allowed"


def check(dev, x, w, b, dy, eps=1e-5):
    y, dx, dw, db, tx, tw, tb = reference(x, w, b, dy, eps)
    tol = FP32 if x.dtype == torch.float32 else BF16
    xd = x.to(dev).requires_grad_()
    wd = None if w is None else w.to(dev).requires_grad_()
    bd = None if b is None else b.to(dev).requires_grad_()
    out = layer_norm(xd, wd, bd, eps=eps)
    assert out.dtype == x.dtype
    close(out.detach(), y, tol, "y")
    with torch.no_grad():
        assert torch.equal(layer_norm(xd, wd, bd, eps=eps), out)
    leaves = [t for t in (xd, wd, bd) if t is not None]
    grads = list(torch.autograd.grad(out, leaves, dy.to(dev)))
    close(grads.pop(0), dx, tol, "grad_x", tx)
    for t, want, terms, what in ((w, dw, tw, "grad_weight"), (b, db, tb, "grad_bias")):
        if t is not None:
            got = grads.pop(0).double().cpu()
            # (each term's xh is off by FP32 of its own)
            assert ((got - want).abs() <= (SUMS + FP32) * terms + 1e-12).all(), what


# Rows of one element to rows past the registers, on and off whole 16-byte units.
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [1, 2, 7, 8, 50, 63, 64, 65, 256, 400, 511, 513, 1000, 1024, 1025, 2048, 4095, 4096, 4100,
                               8192, 10001, 16384, 16385, 20000])
def test_row_lengths(dev, D, dtype):
    check(dev, *make((5, D), dtype, seed=D))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 256), (3, 64), (4, 65), (257, 40), (2, 700, 400), (3, 5, 7, 33), (5000, 16), (40, 17000)])
def test_rows(dev, shape, dtype):
    check(dev, *make(shape, dtype, seed=1))


@pytest.mark.gpu
def test_without_parameters(dev):
    x, w, b, dy = make((30, 100))
    check(dev, x, None, None, dy)
    check(dev, x, w, None, dy)
    check(dev, x, None, b, dy)
    check(dev, x, w, b, dy, eps=0.5)


@pytest.mark.gpu
def test_large_mean(dev):
    """A mean a thousand times the spread: the second sum keeps the variance (x itself is exact in fp32)."""
    x = 1024.0 + torch.randint(-8, 9, (20, 512), generator=torch.Generator().manual_seed(0)) / 8.0
    y = reference(x, None, None, x, 1e-5)[0]
    # the mean's own rounding, 26 2^-24 1024 at worst, against a spread of 0.6
    close(layer_norm(x.to(dev)), y, 26 * 2.0 ** -24 * 1024 / 0.6, "y")


@pytest.mark.gpu
def test_constant_and_extreme_rows(dev):
    x = torch.zeros(4, 96)
    x[1] = 3.0
    x[2] = 1e18 * torch.randn(96, generator=torch.Generator().manual_seed(1))
    x[3] = 1e-18 * torch.randn(96, generator=torch.Generator().manual_seed(2))
    y = reference(x, None, None, x, 1e-5)[0]
    got = layer_norm(x.to(dev)).cpu()
    assert (got[:2] == 0).all()
    close(got[2:], y[2:], FP32, "y")
    bad = x.clone()
    bad[1, 5] = float("nan")
    bad[3, 7] = float("inf")
    got = layer_norm(bad.to(dev)).cpu()
    assert torch.isnan(got[1]).all() and torch.isnan(got[3]).any() and torch.isfinite(got[[0, 2]]).all()


@pytest.mark.gpu
def test_layouts(dev):
    x, w, b, dy = (t.to(dev) for t in make((6, 40, 96), torch.bfloat16))
    want = layer_norm(x, w, b)
    wide = torch.zeros(6, 40, 101, dtype=x.dtype, device=dev)
    wide[..., 2:98] = x
    for other in (x.transpose(0, 1).contiguous().transpose(0, 1), wide[..., 2:98], x.flip(-1).contiguous().flip(-1),
                  torch.stack([x, x], -1)[..., 0]):
        assert torch.equal(layer_norm(other, w, b), want)
    assert torch.equal(layer_norm(x[:, :, None].expand(6, 40, 3, 96), w, b)[:, :, 2], want)
    out = x.clone()
    y, mean, rstd = layer_norm_forward(out, w, b, out=out)
    assert y is out and torch.equal(out, want) and mean.shape == rstd.shape == (6, 40)
    gx = layer_norm_backward(dy, x, mean, rstd, w)
    strided = dy.transpose(0, 1).contiguous().transpose(0, 1)
    assert all(torch.equal(p, q) for p, q in zip(gx, layer_norm_backward(strided, wide[..., 2:98], mean, rstd, w)))
    one = dy[:1, :1].expand(6, 40, 96)
    assert all(torch.equal(p, q) for p, q in zip(layer_norm_backward(one, x, mean, rstd, w),
                                                 layer_norm_backward(one.contiguous(), x, mean, rstd, w)))


@pytest.mark.gpu
def test_needs_and_types(dev):
    x, w, b, dy = (t.to(dev) for t in make((50, 80)))
    _, mean, rstd = layer_norm_forward(x, w, b)
    whole = layer_norm_backward(dy, x, mean, rstd, w)
    for need in ((True, False, False), (False, True, False), (False, False, True), (False, True, True)):
        part = layer_norm_backward(dy, x, mean, rstd, w, need_x=need[0], need_weight=need[1], need_bias=need[2])
        for p, q, n in zip(part, whole, need):
            assert torch.equal(p, q) if n else p is None
    half = x.half().requires_grad_()
    wide = w.bfloat16().requires_grad_()
    y = layer_norm(half, wide, b)
    assert y.dtype == torch.float32
    gx, gw = torch.autograd.grad(y, (half, wide), dy)
    assert gx.dtype == torch.float16 and gw.dtype == torch.bfloat16


@pytest.mark.gpu
def test_gradients_against_differences(dev):
    """Central differences of the kernel's forward: h = 2^-6, truncation about
    h^2 times the third derivative, rounding 2^-24 sqrt(n) / h."""
    x, w, b, dy = (t.to(dev) for t in make((40, 50), seed=4))
    _, mean, rstd = layer_norm_forward(x, w, b)
    grads = layer_norm_backward(dy, x, mean, rstd, w)

    def loss(*t):
        return (layer_norm(*t).double() * dy.double()).sum()

    h, gen = 2.0 ** -6, torch.Generator().manual_seed(0)
    for i, grad in enumerate(grads):
        way = torch.randn(grad.shape, generator=gen).to(dev)
        way /= way.norm()
        up, down = (loss(*(t + s * h * way if j == i else t for j, t in enumerate((x, w, b)))) for s in (1.0, -1.0))
        got = (grad.double() * way.double()).sum().item()
        assert abs((up - down).item() / (2 * h) - got) <= 4 * h * h * grad.norm().item() + 1e-3


@pytest.mark.gpu
def test_empty(dev):
    w = torch.ones(8, device=dev)
    for shape in ((0, 8), (3, 0, 8)):
        x = torch.zeros(shape, device=dev, requires_grad=True)
        wl = w.clone().requires_grad_()
        y = layer_norm(x, wl)
        gx, gw = torch.autograd.grad(y, (x, wl), torch.zeros(shape, device=dev))
        assert y.shape == gx.shape == shape and (gw == 0).all()


@pytest.mark.gpu
def test_same_bits_on_every_run_and_graph(dev):
    x, w, b, dy = (t.to(dev) for t in make((3000, 400), torch.bfloat16))

    def everything():
        y, mean, rstd = layer_norm_forward(x, w, b)
        return (y, *layer_norm_backward(dy, x, mean, rstd, w))

    want = everything()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = everything()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for p, q, r in zip(want, everything(), held):
            assert torch.equal(p, q) and torch.equal(p, r)


@pytest.mark.gpu
def test_refusals(dev):
    x = torch.zeros(4, 8, device=dev)
    for bad in (lambda: layer_norm(torch.zeros((), device=dev)), lambda: layer_norm(torch.zeros(3, 0, device=dev)),
                lambda: layer_norm([1.0]), lambda: layer_norm(x, torch.ones(7, device=dev)),
                lambda: layer_norm(x, None, 0.5), lambda: layer_norm_forward(x, out=torch.zeros(4, 9, device=dev)),
                lambda: layer_norm_backward(x[:3], x, x[:, 0], x[:, 0]), lambda: layer_norm_backward(x, x, x[:2, 0], x[:, 0])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="ROCm GPU only"):
        layer_norm(torch.zeros(4, 8))
    from orthossm_amd._native import OsmError
    with pytest.raises(OsmError):
        layer_norm(x, eps=-1.0)
