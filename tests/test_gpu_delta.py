"""The gated delta rule against its float64 token loop (oracle/delta.py).

Tolerances.  Everything is fp32 arithmetic: a result passes about six products
in turn (scores, triangular system, state read, output, and in the backward as
many again), each a sum of up to 128 terms whose rounding adds to about
sqrt(128) 2^-24 of the result's norm at worst, and products of up to S/64 state
maps whose errors do not grow (every map shrinks the state or keeps its norm):
12 sqrt(128) 2^-24 = 8e-6 of a result's norm.  bf16 results add one rounding
to nearest, at most 2^-8 of each element (8 significant bits).  dL/dg and dL/dbeta are sums of
such results with cancellation, so they get twice the fp32 bound.
"""
import math

import pytest
import torch

from oracle import delta as O
from orthossm_amd import gated_delta, gated_delta_backward, gated_delta_forward, gated_delta_step

FP32 = 8e-6
BF16 = 2.0 ** -8 + FP32


def make(B, S, H, dk, dv=None, Hk=None, dtype=torch.float32, seed=0, decay=0.1, beta_max=1.0, same_keys=False):
    gen = torch.Generator().manual_seed(seed)
    dv, Hk = dv or dk, Hk or H

    def rand(*shape):
        return torch.randn(*shape, generator=gen)

    q, k = (torch.nn.functional.normalize(rand(B, S, Hk, dk), dim=-1) for _ in range(2))
    if same_keys:
        k = k[:, :1].expand(B, S, Hk, dk).clone()
    return dict(q=q.to(dtype), k=k.to(dtype), v=rand(B, S, H, dv).to(dtype), g=-decay * torch.rand(B, S, H, generator=gen),
                beta=beta_max * torch.sigmoid(rand(B, S, H)), state_init=0.5 * rand(B, H, dk, dv),
                grad_out=rand(B, S, H, dv).to(dtype), grad_state=rand(B, H, dk, dv))


def on(t, dev):
    return {n: x.to(dev) if isinstance(x, torch.Tensor) else x for n, x in t.items()}


def args(t):
    return [t[n] for n in ("q", "k", "v", "g", "beta")]


def close(got, want, tol, what):
    got, want = got.double().cpu(), want.double()
    assert got.shape == want.shape, what
    assert torch.isfinite(got).all(), f"{what}: not finite"
    err, size = (got - want).norm().item(), want.norm().item()
    assert err <= tol * size + 1e-30, f"{what}: {err / (size + 1e-300):.2e} of the norm, {tol:.1e} allowed"


def check_forward(dev, t, lengths=None, **kw):
    want, fin = O.gated_delta(*args(t), state_init=t["state_init"], lengths=lengths, **kw)
    d = on(t, dev)
    got, state = gated_delta_forward(*args(d), state_init=d["state_init"], return_state=True,
                                     lengths=None if lengths is None else lengths.to(dev), **kw)
    assert got.dtype == t["v"].dtype
    close(got, want, FP32 if t["v"].dtype == torch.float32 else BF16, "out")
    close(state, fin, FP32, "state")


def check_train(dev, t, lengths=None, init=True, **kw):
    more = dict(state_init=t["state_init"]) if init else {}
    want = O.gated_delta_grads(*args(t), t["grad_out"], t["grad_state"], lengths=lengths, **more, **kw)
    d = on(t, dev)
    leaves = [x.requires_grad_() for x in args(d)] + ([d["state_init"].requires_grad_()] if init else [])
    out, fin = gated_delta(*args(d), state_init=d["state_init"] if init else None, return_state=True,
                           lengths=None if lengths is None else lengths.to(dev), **kw)
    grads = torch.autograd.grad((out, fin), leaves, (d["grad_out"], d["grad_state"]))
    names = ("out", "state", "grad_q", "grad_k", "grad_v", "grad_g", "grad_beta", "grad_init")
    for name, got, ref in zip(names, (out, fin, *grads), want):
        wide = got.dtype == torch.float32
        close(got, ref, (2 * FP32 if name in ("grad_g", "grad_beta") else FP32) if wide else BF16, name)


# One token to several chunks, around every boundary; head sizes on and off
# the 16- and 64-wide blocks, equal and unequal, shared heads.
@pytest.mark.gpu
@pytest.mark.parametrize("S", [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 200])
def test_lengths(dev, S):
    check_forward(dev, make(2, S, 2, 32, seed=S))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,Hk,dk,dv", [(1, 1, 1, 1), (2, 2, 16, 16), (4, 2, 24, 40), (2, 1, 50, 50), (2, 2, 64, 64),
                                        (3, 1, 80, 33), (2, 1, 65, 65), (1, 1, 128, 128), (4, 2, 100, 16), (1, 1, 16, 200)])
def test_heads_and_types(dev, H, Hk, dk, dv, dtype):
    check_forward(dev, make(2, 150, H, dk, dv, Hk, dtype, seed=dk + dv))
    check_forward(dev, make(2, 9, H, dk, dv, Hk, dtype, seed=dk + dv + 1))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("S,H,Hk,dk,dv", [(1, 1, 1, 8, 8), (64, 2, 2, 32, 32), (130, 2, 1, 50, 50), (100, 4, 2, 24, 40),
                                          (129, 2, 2, 64, 64), (70, 2, 2, 65, 33), (200, 2, 1, 128, 128),
                                          (100, 3, 1, 80, 130)])
def test_gradients(dev, S, H, Hk, dk, dv, dtype):
    check_train(dev, make(2, S, H, dk, dv, Hk, dtype, seed=S))
    check_train(dev, make(2, S, H, dk, dv, Hk, dtype, seed=S + 1), init=False, scale=0.7)


@pytest.mark.gpu
def test_long_rows(dev):
    check_forward(dev, make(1, 2500, 2, 16, decay=0.01))
    check_train(dev, make(1, 1000, 1, 32, decay=0.01))


# Rows of different lengths, an empty one among them, NaN and infinities where
# the mask says that nothing is.
@pytest.mark.gpu
@pytest.mark.parametrize("S", [5, 70, 200])
def test_row_lengths(dev, S):
    lengths = torch.tensor([S, 0, 1, S // 2, S + 7], dtype=torch.int32)
    t = make(5, S, 2, 24, 40, 1, seed=S)
    check_forward(dev, t, lengths)
    check_train(dev, make(5, S, 2, 24, 40, 1, seed=S), lengths)
    bad = {n: x.clone() for n, x in t.items()}
    for b, n in enumerate(lengths.tolist()):
        for name, value in (("q", math.nan), ("k", math.inf), ("v", -math.inf), ("g", math.nan), ("beta", math.inf),
                            ("grad_out", math.nan)):
            bad[name][b, n:] = value
    for x, y in zip(_all(dev, t, lengths), _all(dev, bad, lengths)):
        assert torch.equal(x, y)


def _all(dev, t, lengths):
    d = on(t, dev)
    out, fin = gated_delta_forward(*args(d), state_init=d["state_init"], lengths=lengths.to(dev), return_state=True)
    grads = gated_delta_backward(*args(d), d["grad_out"], state_init=d["state_init"], lengths=lengths.to(dev),
                                 grad_state=d["grad_state"], need_init=True)
    return (out, fin, *grads)


@pytest.mark.gpu
def test_lengths_of_other_whole_types(dev):
    t = on(make(3, 40, 1, 16), dev)
    want = gated_delta_forward(*args(t), lengths=torch.tensor([40, 0, 7], dtype=torch.int32, device=dev))
    for lengths in (torch.tensor([1 << 40, -5, 7]), torch.tensor([40, 0, 7], dtype=torch.int16)):
        assert torch.equal(gated_delta_forward(*args(t), lengths=lengths), want)


# Gates at their ends: no decay, a full reset, beta 0, 1 and above; equal keys,
# where the triangular system is as far from the identity as it gets.
@pytest.mark.gpu
@pytest.mark.parametrize("decay", [0.0, 1.0, 30.0])
@pytest.mark.parametrize("beta_max", [0.0, 1.0, 1.9])
def test_gates(dev, decay, beta_max):
    check_forward(dev, make(1, 150, 2, 32, decay=decay, beta_max=beta_max))
    check_train(dev, make(1, 150, 2, 32, decay=decay, beta_max=beta_max))


@pytest.mark.gpu
def test_equal_keys(dev):
    t = make(1, 130, 2, 32, same_keys=True)
    t["beta"] = torch.ones_like(t["beta"])
    check_forward(dev, t)
    check_train(dev, t)


@pytest.mark.gpu
@pytest.mark.parametrize("S", [10, 100])
def test_reset(dev, S):
    """g = -inf: the state is forgotten; what comes after does not see it."""
    t = make(1, S, 2, 32)
    t["g"][:, S // 2] = -math.inf
    check_forward(dev, t)
    late = {n: x[:, S // 2:] if n in ("q", "k", "v", "g", "beta") else x for n, x in t.items()}
    want, fin = O.gated_delta(*args(late))
    d = on(t, dev)
    out, state = gated_delta_forward(*args(d), state_init=d["state_init"], return_state=True)
    close(out[:, S // 2:], want, FP32, "out after the reset")
    close(state, fin, FP32, "state")


@pytest.mark.gpu
def test_strides(dev):
    """Head-major and padded layouts, rows off 4-element boundaries, gates of
    any order, expanded heads: the same bits as contiguous tensors."""
    t = on(make(2, 100, 2, 32), dev)
    want = gated_delta_forward(*args(t), return_state=True)
    head_major = {n: t[n].transpose(1, 2).contiguous().transpose(1, 2) for n in ("q", "k", "v", "g", "beta")}
    padded = {n: torch.nn.functional.pad(t[n], (1, 2))[..., 1:33] for n in ("q", "k", "v")}
    reversed_lanes = {n: t[n].flip(-1).contiguous().flip(-1) for n in ("q", "k", "v")}
    strided = {n: torch.stack([t[n], -t[n]], -1)[..., 0] for n in ("q", "k", "v")}
    for other in (head_major, padded, reversed_lanes, strided):
        got = gated_delta_forward(*args({**t, **other}), return_state=True)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    one = {**t, "q": t["q"][:, :, :1].expand(2, 100, 2, 32), "beta": t["beta"][:, :1].expand(2, 100, 2)}
    same = {**one, "q": one["q"].contiguous(), "beta": one["beta"].contiguous()}
    assert torch.equal(gated_delta_forward(*args(one)), gated_delta_forward(*args(same)))


@pytest.mark.gpu
def test_gradients_of_broadcast_inputs(dev):
    t = make(2, 90, 2, 16)
    wide = dict(t, q=t["q"][:, :, :1].expand(2, 90, 2, 16), beta=t["beta"][:, :1].expand(2, 90, 2))
    want = O.gated_delta_grads(*args(wide), t["grad_out"], None, state_init=t["state_init"])
    d = on(t, dev)
    q1, b1 = d["q"][:, :, :1].contiguous().requires_grad_(), d["beta"][:, :1].contiguous().requires_grad_()
    out = gated_delta(q1.expand(2, 90, 2, 16), d["k"], d["v"], d["g"], b1.expand(2, 90, 2), state_init=d["state_init"])
    gq, gb = torch.autograd.grad(out, (q1, b1), d["grad_out"])
    close(gq, want[2].sum(2, keepdim=True), FP32, "grad_q")
    close(gb, want[6].sum(1, keepdim=True), 2 * FP32, "grad_beta")


@pytest.mark.gpu
def test_gradients_against_differences(dev):
    """Central differences of the kernel's own forward, along a random
    direction of every input: h = 2^-7 leaves a truncation of about h^2 and a
    rounding of 2^-24 sqrt(n) / h of a sum of n outputs of order one."""
    t = on(make(1, 80, 2, 16, seed=3), dev)
    names = ("q", "k", "v", "g", "beta", "state_init")
    grads = gated_delta_backward(*args(t), t["grad_out"], state_init=t["state_init"], grad_state=t["grad_state"],
                                 need_init=True)

    def loss(u):
        out, fin = gated_delta_forward(*args(u), state_init=u["state_init"], return_state=True)
        return (out.double() * t["grad_out"].double()).sum() + (fin.double() * t["grad_state"].double()).sum()

    h = 2.0 ** -7
    gen = torch.Generator().manual_seed(1)
    for name, grad in zip(names, grads):
        way = torch.randn(t[name].shape, generator=gen).to(dev)
        way /= way.norm()
        up, down = (loss({**t, name: t[name] + s * h * way}) for s in (1.0, -1.0))
        want = ((up - down) / (2 * h)).item()
        got = (grad.double() * way.double()).sum().item()
        assert abs(got - want) <= 4 * h * h * grad.norm().item() + 1e-3, name


# Serving: one token a row, the same as a sequence cut into tokens.
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,H,Hk,dk,dv", [(1, 8, 8, 64, 64), (3, 2, 1, 33, 50), (2, 4, 2, 128, 128), (5, 1, 1, 1, 1),
                                          (2, 2, 2, 16, 100)])
def test_step(dev, B, H, Hk, dk, dv, dtype):
    T = 5
    t = make(B, T, H, dk, dv, Hk, dtype, seed=B)
    want, fin = O.gated_delta(*args(t), state_init=t["state_init"])
    d = on(t, dev)
    state = d["state_init"].clone()
    outs = [gated_delta_step(*(d[n][:, i] for n in ("q", "k", "v", "g", "beta")), state) for i in range(T)]
    close(torch.stack(outs, 1), want, FP32 if dtype == torch.float32 else BF16, "out")
    close(state, fin, FP32, "state")


@pytest.mark.gpu
def test_step_slots(dev):
    """Rows at scattered slots of a strided pool, idle ones, and one past it."""
    B, H, dk, dv = 6, 2, 32, 40
    t = on(make(B, 1, H, dk, dv), dev)
    one = [t[n][:, 0] for n in ("q", "k", "v", "g", "beta")]
    pool = torch.randn(9, 2, H, dk, dv, device=dev)[:, 0]
    before = pool.clone()
    slots = torch.tensor([7, -1, 0, 3, -9, 9], device=dev)
    out = gated_delta_step(*one, pool, slots=slots)
    live = [0, 2, 3]
    want_state = before[slots[live]].clone()
    want = gated_delta_step(*(x[live].contiguous() for x in one), want_state)
    assert torch.equal(out[live], want) and torch.equal(pool[slots[live]], want_state)
    rest = [i for i in range(9) if i not in (7, 0, 3)]
    assert torch.equal(pool[rest], before[rest])
    assert (out[[1, 4]] == 0).all() and torch.isnan(out[5]).all()


@pytest.mark.gpu
def test_state_past_32_bits(dev):
    """A pool whose last slot starts past 2^31 elements."""
    H, dk, dv = 16, 128, 128
    n = (1 << 31) // (H * dk * dv) + 2
    pool = torch.empty(n, H, dk, dv, device=dev)
    t = on(make(2, 1, H, dk, dv), dev)
    one = [t[x][:, 0] for x in ("q", "k", "v", "g", "beta")]
    slots = torch.tensor([n - 1, 1], device=dev)
    pool[slots] = t["state_init"]
    out = gated_delta_step(*one, pool, slots=slots)
    small = t["state_init"].clone()
    want = gated_delta_step(*one, small)
    assert torch.equal(out, want) and torch.equal(pool[slots], small)


@pytest.mark.gpu
def test_sequence_continues_from_a_state(dev):
    """A sequence in pieces, chunks, tokens and all, is the whole sequence."""
    t = make(2, 200, 2, 32)
    want, fin = O.gated_delta(*args(t), state_init=t["state_init"])
    d = on(t, dev)
    state, outs = d["state_init"].clone(), []
    for lo, hi in ((0, 70), (70, 71), (71, 80), (80, 200)):
        piece = [d[n][:, lo:hi] for n in ("q", "k", "v", "g", "beta")]
        out, same = gated_delta_forward(*piece, state_init=state, return_state=True, state_out=state)
        assert same is state
        outs.append(out)
    close(torch.cat(outs, 1), want, FP32, "out")
    close(state, fin, FP32, "state")


@pytest.mark.gpu
def test_empty(dev):
    t = on(make(2, 0, 2, 16), dev)
    out, fin = gated_delta_forward(*args(t), state_init=t["state_init"], return_state=True)
    assert out.shape == (2, 0, 2, 16) and torch.equal(fin, t["state_init"])
    out, fin = gated_delta_forward(*args(t), return_state=True)
    assert (fin == 0).all()
    grads = gated_delta_backward(*args(t), t["grad_out"], grad_state=t["grad_state"], need_init=True)
    assert torch.equal(grads[5], t["grad_state"])
    none = on(make(0, 5, 2, 16), dev)
    assert gated_delta_forward(*args(none)).shape == (0, 5, 2, 16)
    assert gated_delta_step(*(none[n][:, 0] for n in ("q", "k", "v", "g", "beta")), none["state_init"]).shape == (0, 2, 16)


@pytest.mark.gpu
def test_same_bits_on_every_run_stream_and_graph(dev):
    t = on(make(2, 300, 4, 64, Hk=2, dtype=torch.bfloat16), dev)

    def everything():
        out, fin = gated_delta_forward(*args(t), state_init=t["state_init"], return_state=True)
        return (out, fin, *gated_delta_backward(*args(t), t["grad_out"], state_init=t["state_init"],
                                                grad_state=t["grad_state"], need_init=True))

    want = everything()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = everything()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = everything()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        again = everything()
        for x, y, z, w in zip(want, other, held, again):
            assert torch.equal(x, y) and torch.equal(x, z) and torch.equal(x, w)


@pytest.mark.gpu
def test_partial_gradients_and_mixed_types(dev):
    t = make(1, 70, 2, 16, seed=9)
    t["q"] = t["q"].bfloat16()          # with fp32 k and v: fp32 arithmetic, q's gradient in q's type
    want = O.gated_delta_grads(*args(t), t["grad_out"])
    d = on(t, dev)
    d["q"].requires_grad_()
    d["beta"] = d["beta"].double().requires_grad_()
    out = gated_delta(*args(d))
    assert out.dtype == torch.float32
    out.backward(d["grad_out"])
    assert d["q"].grad.dtype == torch.bfloat16 and d["beta"].grad.dtype == torch.float64 and d["k"].grad is None
    close(d["q"].grad, want[2], BF16, "grad_q")
    close(d["beta"].grad, want[6], 2 * FP32, "grad_beta")


@pytest.mark.gpu
def test_refusals(dev):
    t = on(make(2, 8, 4, 16, Hk=2), dev)
    ok = args(t)

    def refuses(error, *a, **kw):
        with pytest.raises(error):
            gated_delta_forward(*a, **kw)

    refuses(RuntimeError, *(x.cpu() for x in ok))
    refuses(ValueError, ok[0][0], *ok[1:])                                    # not [B,S,heads,size]
    refuses(ValueError, ok[0][:, :7], *ok[1:])
    refuses(ValueError, ok[0], ok[1][..., :8], *ok[2:])
    refuses(ValueError, *ok[:2], ok[2][:, :, :3], *ok[3:])                    # heads no multiple of two
    refuses(ValueError, *ok[:3], ok[3][:, :, :2], ok[4])
    refuses(ValueError, *ok[:4], 0.5)
    refuses(ValueError, *ok, state_init=t["state_init"][:1])
    refuses(ValueError, *ok, lengths=torch.ones(2, device=dev))
    refuses(ValueError, *ok, lengths=torch.ones(3, dtype=torch.int32, device=dev))
    refuses(ValueError, *ok, out=torch.empty(2, 8, 4, 16, device=dev, dtype=torch.bfloat16))
    refuses(ValueError, *ok, state_out=torch.empty(2, 4, 16, 16, device=dev).transpose(2, 3))
    wide = torch.zeros(1, 4, 1, 129, device=dev)
    refuses(ValueError, wide, wide, torch.zeros(1, 4, 1, 8, device=dev), *(torch.zeros(1, 4, 1, device=dev),) * 2)
    with pytest.raises(ValueError):
        gated_delta_backward(*ok, t["grad_out"][:, :7])
    one = [x[:, 0] for x in ok]
    pool = t["state_init"]
    for kw in (dict(slots=torch.zeros(2, dtype=torch.int32, device=dev)), dict(slots=torch.zeros(3, dtype=torch.int64, device=dev)),
               dict(slots=torch.zeros(2, dtype=torch.int64)), dict(out=torch.empty(2, 4, 15, device=dev))):
        with pytest.raises(ValueError):
            gated_delta_step(*one, pool, **kw)
    for bad in (pool[:1], pool.double(), pool.transpose(2, 3), pool[0], pool.cpu()):
        with pytest.raises(ValueError):
            gated_delta_step(*one, bad)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,S", [(torch.int8, 130), (torch.uint8, 300), (torch.int16, 33000)])
def test_lengths_of_narrow_types(dev, dtype, S):
    t = on(make(2, S, 1, 4), dev)
    want = gated_delta_forward(*args(t), lengths=torch.tensor([120, 3], dtype=torch.int32, device=dev))
    assert torch.equal(gated_delta_forward(*args(t), lengths=torch.tensor([120, 3], dtype=dtype, device=dev)), want)
