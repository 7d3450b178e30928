"""The global gradient norm and clipping against float64.

Tolerances.  The squares are exact in double and their sums off by far less
than fp32's last bit, so the norm is right to one rounding, 2^-24 (doubled
here), and a scaled element to that of the factor and its own: 2^-23 for fp32,
2^-8 for bf16 on top.
"""
import math

import pytest
import torch

from orthossm_amd import clip_grad_norm, grad_norm

SHAPES = [(1,), (3,), (8192,), (8193,), (129, 65), (4096, 40), (0,), (2, 0, 3), (), (77,), (1000, 3, 7)]


def make(dev, shapes=SHAPES, dtypes=(torch.float32, torch.bfloat16), size=0.1, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return [(size * torch.randn(s, generator=gen)).to(dtypes[i % len(dtypes)]).to(dev) for i, s in enumerate(shapes)]


def norm_of(grads):
    return math.sqrt(sum(t.double().square().sum().item() for t in grads))


def check(grads, max_norm, eps=1e-6):
    before = [t.clone() for t in grads]
    want = norm_of(before)
    norm = clip_grad_norm(grads, max_norm, eps=eps)
    assert norm.shape == () and norm.dtype == torch.float32
    assert abs(norm.item() - want) <= 2.0 ** -23 * want
    factor = min(1.0, max_norm / (want + eps))
    for t, b in zip(grads, before):
        ref = b.double() * factor
        tol = 2.0 ** -23 + (2.0 ** -8 if t.dtype == torch.bfloat16 else 0.0)
        assert ((t.double() - ref).abs() <= tol * ref.abs() + 1e-40).all()
    return before


@pytest.mark.gpu
@pytest.mark.parametrize("dtypes", [(torch.float32,), (torch.bfloat16,), (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("max_norm", [1.0, 1e-3, 0.0])
def test_clip(dev, dtypes, max_norm):
    check(make(dev, dtypes=dtypes), max_norm)


@pytest.mark.gpu
def test_within_the_limit_nothing_changes(dev):
    grads = make(dev)
    before = check(grads, 1e6)
    assert all(torch.equal(t, b) for t, b in zip(grads, before))
    assert torch.equal(grad_norm(grads), clip_grad_norm(grads, 1e6))


@pytest.mark.gpu
@pytest.mark.parametrize("count", [1, 149, 150, 151, 700])
def test_many_tensors(dev, count):
    """More than one launch holds, of sizes off every alignment."""
    grads = make(dev, [((i * 37) % 301,) for i in range(count - 1)] + [(40000,)])
    check(grads, 0.5)
    assert abs(grad_norm(grads).item() - norm_of(grads)) <= 2.0 ** -23 * norm_of(grads)


@pytest.mark.gpu
def test_unaligned_views_and_layouts(dev):
    flat = torch.randn(50000, device=dev)
    half = torch.randn(50000, device=dev).bfloat16()
    kept = flat.clone(), half.clone()
    grads = [flat[1:20000], half[3:9001], flat[20001:45001].view(100, 250).t(), flat[45002:49002].view(20, 200)[:, ::2],
             half[10000:42768].view(2, 128, 128).permute(2, 0, 1)]
    check(grads, 1.0)
    assert flat[0] == kept[0][0] and flat[20000] == kept[0][20000] and torch.equal(flat[49002:], kept[0][49002:])
    gap = flat[45002:49002].view(20, 200)[:, 1::2], kept[0][45002:49002].view(20, 200)[:, 1::2]
    assert torch.equal(*gap) and torch.equal(half[:3], kept[1][:3]) and torch.equal(half[9001:10000], kept[1][9001:10000])


@pytest.mark.gpu
def test_range(dev):
    """Squares past fp32's range at both ends."""
    for size in (1e25, 1e-30):
        grads = make(dev, [(1000,), (50, 3)], (torch.float32,), size)
        assert abs(grad_norm(grads).item() - norm_of(grads)) <= 2.0 ** -23 * norm_of(grads)
    check(make(dev, [(1000,)], (torch.float32,), 1e25), 1.0)


@pytest.mark.gpu
def test_nan_and_infinity(dev):
    for bad, others in ((math.nan, "nan"), (math.inf, "zero")):
        grads = make(dev, [(500,), (40, 40)])
        grads[1][3, 3] = bad
        norm = clip_grad_norm(grads, 1.0)
        rest = torch.cat([t.flatten().float() for t in grads])
        assert not torch.isfinite(norm)
        assert torch.isnan(grads[1][3, 3])
        assert (torch.isnan(rest) if others == "nan" else (rest == 0)).sum() >= rest.numel() - 1


@pytest.mark.gpu
def test_none_and_empty(dev):
    empty = torch.zeros(0, device=dev)
    assert clip_grad_norm([empty, empty], 1.0).item() == 0.0 and grad_norm(empty).item() == 0.0
    zero = torch.zeros(10, device=dev)
    assert clip_grad_norm(zero, 1.0).item() == 0.0 and (zero == 0).all()


@pytest.mark.gpu
def test_same_bits_on_every_run_and_graph(dev):
    """Also with the sizes that several workgroups share."""
    first = make(dev, [(3000, 700), (5,), (1 << 20,)])
    want = [t.clone() for t in first]
    norm = clip_grad_norm(want, 1.0)
    held = [t.clone() for t in first]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held_norm = clip_grad_norm(held, 1.0)
    for _ in range(3):
        for t, f in zip(held, first):
            t.copy_(f)
        graph.replay()
        torch.cuda.synchronize()
        again = [t.clone() for t in first]
        assert torch.equal(clip_grad_norm(again, 1.0), norm) and torch.equal(held_norm, norm)
        assert all(torch.equal(a, w) and torch.equal(h, w) for a, h, w in zip(again, held, want))


@pytest.mark.gpu
def test_refusals(dev):
    x = torch.ones(4, device=dev)
    for error, grads in ((ValueError, []), (ValueError, [1.0]), (RuntimeError, [torch.ones(4)]), (TypeError, [x.double()]),
                         (TypeError, [x.half()]), (ValueError, [x, x]), (ValueError, [x.clone().requires_grad_()])):
        with pytest.raises(error):
            clip_grad_norm(grads, 1.0)
    from orthossm_amd._native import OsmError
    for kw in (dict(max_norm=-1.0), dict(max_norm=math.nan), dict(max_norm=1.0, eps=-1.0)):
        with pytest.raises(OsmError):
            clip_grad_norm([x], **kw)
    assert (x == 1).all()


@pytest.mark.gpu
def test_tensors_that_share_memory_are_refused(dev):
    """Before anything is written; the norm alone takes them."""
    flat = torch.ones(240, device=dev)
    square = flat.view(4, 60)
    for grads in ([flat, flat[1:]], [flat, square.t()], [square[:, ::2], square[:, ::2]], [flat[10:], flat[:3].expand(2, 3)]):
        with pytest.raises(ValueError, match="share memory"):
            clip_grad_norm(grads, 1.0)
        assert (flat == 1).all()
        assert grad_norm(grads).item() == pytest.approx(norm_of(grads))
    clip_grad_norm([square[:, ::2], square[:, 1::2]], 1.0)
    assert abs(norm_of([flat]) - 1.0) <= 1e-5
