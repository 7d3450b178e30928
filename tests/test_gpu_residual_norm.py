"""The residual norm against float64.

Tolerances.  As the layer norm's: a row's sums add at most 16 elements a thread, then
a tree of ten levels, 26 roundings of 2^-24 relative to the row's absolute mean, which
is at most five standard deviations here: 8e-6 of a result's size.  n and every
gradient pass through two norms, so twice that; the gate's e^-|v| is off by at most
|v| 2^-24 and a few units, within it.  bf16 results add half a unit in the last place,
2^-8 of each element.  The parameters' gradients add up to 200 terms in a row (a
thread's rows, four row groups, an eighth of the lines of sums): 200 2^-24 of the sum of
the terms' sizes.  The gradients to rows are differences (for one or two elements a row
nearly all of them cancels), so their bounds are relative to the size of their terms.
"""
import ctypes

import pytest
import torch

from orthossm_amd import _native as nat
from orthossm_amd import block_norm, layer_norm, residual_norm, residual_norm_backward, residual_norm_forward

pytestmark = pytest.mark.gpu
FP32 = 1.6e-5
SUMS = 200 * 2.0 ** -24
NAMES = ("grad_x", "grad_y", "grad_gate", "grad_scale", "grad_weight", "grad_bias")


def eps_of(dtype):
    return 2.0 ** -8 if dtype == torch.bfloat16 else 0.0


def make(shape, stream=torch.float32, block=torch.float32, seed=0):
    gen = torch.Generator().manual_seed(seed)
    D = shape[-1]

    def rand(*s):
        return torch.randn(*s, generator=gen)

    return dict(x=(2 * rand(*shape)).to(stream), y=(rand(*shape) * (0.5 + rand(*shape[:-1], 1).abs()) + rand(*shape[:-1], 1)).to(block),
                gate=rand(*shape).to(block), scale=0.5 + 0.2 * rand(D), weight=1 + 0.3 * rand(D), bias=0.3 * rand(D),
                grad_r=rand(*shape).to(stream), grad_n=rand(*shape).to(block))


def reference(t, norm_y=True, rms=False, eps=1e-5):
    """(r, n), the gradients, and the sizes of the gradients' terms."""
    d = {k: None if v is None else v.double() for k, v in t.items()}
    x, y, gate = d["x"], d["y"], d["gate"]
    one = torch.ones(x.shape[-1], dtype=torch.float64)
    scale, weight = (one if d[k] is None else d[k] for k in ("scale", "weight"))

    def norm(v):
        m = v - v.mean(-1, keepdim=True) if not rms else v
        s = (m.square().mean(-1, keepdim=True) + eps) ** -0.5
        return m * s, s

    def back(g, vh, s, sizes):
        mean = (lambda v: v.abs().mean(-1, keepdim=True)) if sizes else (lambda v: v.mean(-1, keepdim=True))
        a, b = (0 if rms else mean(g)), mean(g * vh)
        return s * (g.abs() + a + vh.abs() * b) if sizes else s * (g - a - vh * b)

    yh, sy = norm(y) if norm_y else (y, 1.0)
    o = torch.sigmoid(gate) if gate is not None else torch.ones_like(y)
    rest = torch.sigmoid(-gate) if gate is not None else torch.zeros_like(y)
    r = x + scale * o * yh
    rh, sr = norm(r)
    n = rh * weight + (0 if d["bias"] is None else d["bias"])
    zero = torch.zeros_like(x)
    dn, gr = (zero if d[k] is None else d[k] for k in ("grad_n", "grad_r"))
    lead = tuple(range(x.dim() - 1))

    def gradients(sizes):
        # (of the sizes: every sum without its signs)
        mag = torch.abs if sizes else (lambda v: v)
        dr = mag(gr) + back(mag(dn * weight), mag(rh), sr, sizes)
        du = dr * mag(scale)
        e = du * o
        dy = back(e, mag(yh), sy, sizes) if norm_y else e
        return dr, dy, e * mag(yh) * rest, (dr * mag(yh) * o).sum(lead), mag(dn * rh).sum(lead), mag(dn).sum(lead)

    return (r, n), gradients(False), gradients(True)


def close(got, want, tol, what, terms=None):
    got = got.double().cpu()
    assert got.shape == want.shape and torch.isfinite(got).all(), what
    err, size = (got - want).norm().item(), (want if terms is None else terms).norm().item()
    assert err <= tol * size + 1e-12, f"{what}: {err / (size + 1e-300):.2e} of the norm, {tol:.1e} allowed"


def check(dev, t, **form):
    outs, grads, sizes = reference(t, **form)
    d = {k: None if v is None else v.to(dev) for k, v in t.items()}
    names = [k for k in ("x", "y", "gate", "scale", "weight", "bias") if d[k] is not None]
    for k in names:
        d[k].requires_grad_()
    call = dict(gate=d["gate"], scale=d["scale"], **form)
    r, n = residual_norm(d["x"], d["y"], d["weight"], d["bias"], **call)
    es, eb = eps_of(t["x"].dtype), eps_of(t["y"].dtype)
    assert r.dtype == t["x"].dtype and n.dtype == t["y"].dtype
    close(r.detach(), outs[0], FP32 + es, "r")
    close(n.detach(), outs[1], FP32 + eb, "n")
    with torch.no_grad():
        assert all(torch.equal(p, q) for p, q in zip(residual_norm(d["x"], d["y"], d["weight"], d["bias"], **call), (r, n)))
    outs = [(o, g) for o, g in ((r, d["grad_r"]), (n, d["grad_n"])) if g is not None]
    got = dict(zip(names, torch.autograd.grad([o for o, _ in outs], [d[k] for k in names], [g for _, g in outs], allow_unused=True)))
    for k, want, terms, name in zip(("x", "y", "gate", "scale", "weight", "bias"), grads, sizes, NAMES):
        if k not in got:
            continue
        if k in ("scale", "weight", "bias"):
            # (each term is off by FP32 of its own)
            assert ((got[k].double().cpu() - want).abs() <= (SUMS + 2 * FP32) * terms + 1e-12).all(), name
        else:
            close(got[k], want, 2 * FP32 + (es if k == "x" else eb), name, terms)


TYPES = [(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16)]


# Rows of one element to rows past the registers, on and off whole 16-byte units.
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("D", [1, 2, 7, 8, 50, 63, 64, 65, 128, 256, 400, 511, 513, 1000, 1024, 1025, 2048, 4096, 4100, 8192, 8193,
                               10001, 16384, 16385, 20000])
def test_row_lengths(dev, D, types):
    check(dev, make((5, D), *types, seed=D))


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("norm_y,rms", [(True, True), (False, False), (False, True)])
@pytest.mark.parametrize("D", [1, 33, 200, 1000, 5000, 9000])
def test_norms(dev, D, norm_y, rms, types):
    check(dev, make((7, D), *types, seed=D), norm_y=norm_y, rms=rms)


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("shape", [(1, 256), (3, 64), (257, 40), (2, 700, 400), (3, 5, 7, 33), (5000, 16), (40, 9000)])
def test_rows(dev, shape, types):
    check(dev, make(shape, *types, seed=1))


@pytest.mark.parametrize("without", ["gate", "scale", "weight", "bias", "grad_r", "grad_n", "gate scale weight bias"])
@pytest.mark.parametrize("D", [100, 9000])
def test_without(dev, without, D):
    t = make((30, D), seed=2)
    for k in without.split():
        t[k] = None
    check(dev, t, eps=0.25)


def test_is_the_layer_norm_where_the_block_adds_nothing(dev):
    t = {k: v.to(dev) for k, v in make((40, 300)).items()}
    r, n = residual_norm(t["x"], t["y"], t["weight"], t["bias"], scale=torch.zeros(300, device=dev))
    assert torch.equal(r, t["x"]) and torch.equal(n, layer_norm(t["x"], t["weight"], t["bias"]))


def test_gates_far_out(dev):
    t = make((6, 64))
    t["gate"][0], t["gate"][1], t["gate"][2], t["gate"][3] = float("inf"), -float("inf"), 3e38, -3e38
    d = {k: v.to(dev) for k, v in t.items()}
    r, n, stats = residual_norm_forward(d["x"], d["y"], gate=d["gate"])
    whole = residual_norm(d["x"], d["y"])[0]
    assert torch.equal(r[[0, 2]], whole[[0, 2]]) and torch.equal(r[[1, 3]], d["x"][[1, 3]])
    grads = residual_norm_backward(d["grad_r"], d["grad_n"], d["x"], d["y"], stats, gate=d["gate"])
    assert all(torch.isfinite(g).all() for g in grads) and (grads[2][:4] == 0).all() and (grads[1][[1, 3]] == 0).all()


def test_constant_and_extreme_rows(dev):
    t = make((5, 96), seed=3)
    t["y"][0] = 3.0           # a row without spread: its norm is 0
    t["y"][1] *= 1e15
    t["x"][2], t["y"][2] = 0.0, 0.0
    t["scale"] = t["weight"] = t["bias"] = t["gate"] = None
    (r, n), *_ = reference(t)
    got = residual_norm(t["x"].to(dev), t["y"].to(dev))
    assert torch.equal(got[0][0].cpu(), t["x"][0]) and (got[1][2] == 0).all()
    close(got[0], r, FP32, "r")
    close(got[1], n, FP32, "n")
    t["y"][3, 4] = float("nan")
    got = residual_norm(t["x"].to(dev), t["y"].to(dev))
    assert all(torch.isnan(g[3]).all() and torch.isfinite(g[[0, 1, 2, 4]]).all() for g in got)


def test_layouts(dev):
    t = {k: v.to(dev) for k, v in make((6, 40, 96), torch.float32, torch.bfloat16).items()}
    args, call = (t["weight"], t["bias"]), dict(scale=t["scale"])
    want = residual_norm(t["x"], t["y"], *args, gate=t["gate"], **call)
    wide = torch.zeros(6, 40, 200, dtype=t["y"].dtype, device=dev)
    wide[..., 2:98], wide[..., 98:194] = t["y"], t["gate"]
    turned = t["x"].transpose(0, 1).contiguous().transpose(0, 1)
    for x, y, gate in ((t["x"], wide[..., 2:98], wide[..., 98:194]), (turned, t["y"], t["gate"]),
                       (t["x"].flip(-1).contiguous().flip(-1), t["y"], torch.stack([t["gate"]] * 2, -1)[..., 0])):
        assert all(torch.equal(p, q) for p, q in zip(residual_norm(x, y, *args, gate=gate, **call), want))
    r, n, stats = residual_norm_forward(t["x"], t["y"], *args, gate=t["gate"], **call)
    assert torch.equal(r, want[0]) and torch.equal(n, want[1]) and stats.shape == (6, 40, 4)
    back = residual_norm_backward(t["grad_r"], t["grad_n"], t["x"], t["y"], stats, t["weight"], gate=t["gate"], **call)
    gr = t["grad_r"].transpose(0, 1).contiguous().transpose(0, 1)
    assert all(torch.equal(p, q) for p, q in zip(back, residual_norm_backward(
        gr, wide[..., 2:98] * 0 + t["grad_n"], turned, wide[..., 2:98], stats, t["weight"], gate=wide[..., 98:194], **call)))
    one = t["grad_n"][:1, :1].expand(6, 40, 96)      # a broadcast gradient: strides of zero
    assert all(torch.equal(p, q) for p, q in zip(
        residual_norm_backward(None, one, t["x"], t["y"], stats, t["weight"], gate=t["gate"], **call),
        residual_norm_backward(None, one.contiguous(), t["x"], t["y"], stats, t["weight"], gate=t["gate"], **call)))


def test_needs_and_types(dev):
    t = {k: v.to(dev) for k, v in make((50, 80)).items()}
    _, _, stats = residual_norm_forward(t["x"], t["y"], t["weight"], t["bias"], gate=t["gate"], scale=t["scale"])

    def back(need):
        return residual_norm_backward(t["grad_r"], t["grad_n"], t["x"], t["y"], stats, t["weight"], gate=t["gate"], scale=t["scale"],
                                      need=need)

    whole = back((True,) * 6)
    for i in range(6):
        for need in (tuple(j == i for j in range(6)), tuple(j != i for j in range(6))):
            for p, q, n in zip(back(need), whole, need):
                assert torch.equal(p, q) if n else p is None
    x, y, gate = t["x"].bfloat16().requires_grad_(), t["y"].requires_grad_(), t["gate"].half().requires_grad_()
    scale = t["scale"].double().requires_grad_()
    r, n = residual_norm(x, y, gate=gate, scale=scale)
    assert r.dtype == n.dtype == torch.float32
    grads = torch.autograd.grad((r, n), (x, y, gate, scale), (t["grad_r"], t["grad_n"]))
    assert [g.dtype for g in grads] == [torch.bfloat16, torch.float32, torch.float16, torch.float64]
    for i in range(6):
        mine = [t[k].detach().clone().requires_grad_(j == i) for j, k in enumerate(("x", "y", "gate", "scale", "weight", "bias"))]
        r, n = residual_norm(mine[0], mine[1], mine[4], mine[5], gate=mine[2], scale=mine[3])
        (r.sum() + n.square().sum()).backward()
        assert [m.grad is not None for m in mine] == [j == i for j in range(6)]


def test_gradients_against_differences(dev):
    """Central differences of the kernel's forward, h = 2^-6."""
    t = {k: v.to(dev) for k, v in make((40, 50), seed=4).items()}
    names = ("x", "y", "gate", "scale", "weight", "bias")
    _, _, stats = residual_norm_forward(t["x"], t["y"], t["weight"], t["bias"], gate=t["gate"], scale=t["scale"])
    grads = residual_norm_backward(t["grad_r"], t["grad_n"], t["x"], t["y"], stats, t["weight"], gate=t["gate"], scale=t["scale"])

    def loss(**d):
        r, n = residual_norm(d["x"], d["y"], d["weight"], d["bias"], gate=d["gate"], scale=d["scale"])
        return (r.double() * t["grad_r"].double()).sum() + (n.double() * t["grad_n"].double()).sum()

    h, gen = 2.0 ** -6, torch.Generator().manual_seed(0)
    for k, grad in zip(names, grads):
        way = torch.randn(grad.shape, generator=gen).to(dev)
        way /= way.norm()
        up, down = (loss(**{m: t[m] + s * h * way if m == k else t[m] for m in names}) for s in (1.0, -1.0))
        got = (grad.double() * way.double()).sum().item()
        assert abs((up - down).item() / (2 * h) - got) <= 4 * h * h * grad.norm().item() + 1e-3, k


def test_empty(dev):
    w = torch.ones(8, device=dev)
    for shape in ((0, 8), (3, 0, 8)):
        x = torch.zeros(shape, device=dev, requires_grad=True)
        wl, sl = w.clone().requires_grad_(), w.clone().requires_grad_()
        r, n = residual_norm(x, x.detach(), wl, scale=sl)
        gx, gw, gs = torch.autograd.grad((r, n), (x, wl, sl), (torch.zeros(shape, device=dev),) * 2)
        assert r.shape == n.shape == gx.shape == shape and (gw == 0).all() and (gs == 0).all()


@pytest.mark.parametrize("rows,D", [(70, 33), (300, 1024), (5, 9000), (9, 20000)])
def test_outputs_in_the_inputs_memory(dev, rows, D):
    """From C, r may be x and n may be y."""
    t = {k: v.to(dev) for k, v in make((rows, D), seed=21).items()}
    args = [t[k] for k in ("x", "y", "gate", "scale", "weight", "bias")]
    r, n, _ = residual_norm_forward(args[0], args[1], args[4], args[5], gate=args[2], scale=args[3])
    a, ins, keep = block_norm._prepare(*args, True, False, 1e-5)
    a.r, a.r_stride, a.n, a.n_stride = a.x, a.x_stride, a.y, a.y_stride
    nat.check(nat.load().osm_residual_norm_fwd(ctypes.byref(a), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
    assert torch.equal(t["x"], r) and torch.equal(t["y"], n)


def test_same_bits_on_every_run_and_graph(dev):
    t = {k: v.to(dev) for k, v in make((3000, 400), torch.float32, torch.bfloat16).items()}

    def everything():
        r, n, stats = residual_norm_forward(t["x"], t["y"], t["weight"], t["bias"], gate=t["gate"], scale=t["scale"])
        return (r, n, *residual_norm_backward(t["grad_r"], t["grad_n"], t["x"], t["y"], stats, t["weight"], gate=t["gate"],
                                              scale=t["scale"]))

    want = everything()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = everything()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for p, q, r in zip(want, everything(), held):
            assert torch.equal(p, q) and torch.equal(p, r)


def test_refusals(dev):
    x = torch.zeros(4, 8, device=dev)
    st = torch.zeros(4, 4, device=dev)
    for bad in (lambda: residual_norm(torch.zeros((), device=dev), x), lambda: residual_norm(x, x[:3]), lambda: residual_norm(x, None),
                lambda: residual_norm([1.0], x), lambda: residual_norm(x, x, torch.ones(7, device=dev)),
                lambda: residual_norm(x, x, gate=x[:, :1]), lambda: residual_norm(x, x, scale=0.5),
                lambda: residual_norm(x, x, gate=x.cpu()), lambda: residual_norm(torch.zeros(3, 0, device=dev), torch.zeros(3, 0, device=dev)),
                lambda: residual_norm_backward(x[:3], x, x, x, st), lambda: residual_norm_backward(x, x, x, x, st[:3])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="ROCm GPU only"):
        residual_norm(x.cpu(), x.cpu())
    from orthossm_amd._native import OsmError
    with pytest.raises(OsmError):
        residual_norm(x, x, eps=-1.0)
