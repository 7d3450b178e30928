"""The EMA with a learned gate against float64, token by token.

Tolerances.  A token's decay and its weight are each off by a few units of 2^-24,
and every step rounds the state once more; what is off in one token fades with the
decays, so with o the least weight 1 - a that the gates allow, a state is off by at
most E = 2^-24 (4 / o + 16) of the largest one: twice two errors a step over a memory
of 1 / o steps (the tokens' maps are composed once and run once), and 16 for the
levels of composition.  The adjoint is the same recurrence backward.  dx = o p adds
nothing of size, dgate = a o (h - x) p has the errors of both.  bf16 results add half a
unit in the last place, 2^-8 of the value.
"""
import pytest
import torch

from orthossm_amd import gated_ema, gated_ema_backward, gated_ema_forward, gated_ema_step

pytestmark = pytest.mark.gpu
EPS = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8}


def make(B, S, D, dtype=torch.float32, seed=0, most=6.0):
    gen = torch.Generator().manual_seed(seed)

    def rand(*s):
        return torch.randn(*s, generator=gen)

    x, gate, go = rand(B, S, D).to(dtype), (2.5 + 2.0 * rand(B, S, D)).clamp(max=most).to(dtype), rand(B, S, D).to(dtype)
    return x, gate, rand(B, D), go, rand(B, D)


def reference(x, gate, init, go, gs, lengths=None):
    """h, final, dx, dgate, dinit, and the largest of |h|, |p| and |h - x|."""
    x, a, go = x.double(), torch.sigmoid(gate.double()), go.double()
    o = torch.sigmoid(-gate.double())
    B, S, D = x.shape
    lens = [S] * B if lengths is None else [min(max(int(n), 0), S) for n in lengths]
    out, gx, gg, fin, gi = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x), init.double().clone(), gs.double().clone()
    most = [1e-30, 1e-30, 1e-30]
    for b, n in enumerate(lens):
        h, before = init[b].double(), []
        for t in range(n):
            before.append(h)
            h = a[b, t] * h + o[b, t] * x[b, t]
            out[b, t] = h
        fin[b] = h
        p = gs[b].double()
        for t in reversed(range(n)):
            p = p + go[b, t]
            diff = before[t] - x[b, t]
            gx[b, t], gg[b, t] = o[b, t] * p, a[b, t] * o[b, t] * diff * p
            most = [max(m, v.abs().max().item()) for m, v in zip(most, (h, p, diff))]
            p = a[b, t] * p
        gi[b] = p
    most[0] = max(most[0], out.abs().max().item() if out.numel() else 0.0, init.abs().max().item() if init.numel() else 0.0)
    return out, fin, gx, gg, gi, most


def near(got, want, bound, eps, what):
    got = got.double().cpu()
    assert got.shape == want.shape and torch.isfinite(got).all(), what
    over = (got - want).abs() - eps * want.abs() - bound
    assert not over.numel() or over.max().item() <= 0, f"{what}: {(got - want).abs().max().item():.2e} off, {bound:.2e} allowed"


def check(dev, x, gate, init, go, gs, lengths=None):
    out, fin, gx, gg, gi, (mh, mp, md) = reference(x, gate, init, go, gs, lengths)
    E = 2.0 ** -24 * (4.0 * (1.0 + torch.exp(gate.double().clamp(max=30)).max().item()) + 16.0) if gate.numel() else 0.0
    eps = EPS[x.dtype]
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=dev)
    leaves = [t.to(dev).requires_grad_() for t in (x, gate, init)]
    h, last = gated_ema(leaves[0], leaves[1], state_init=leaves[2], lengths=lens, return_state=True)
    assert h.dtype == x.dtype and last.dtype == torch.float32
    near(h.detach(), out, E * mh, eps, "h")
    near(last.detach(), fin, E * mh, 0.0, "final state")
    grads = torch.autograd.grad((h, last), leaves, (go.to(dev), gs.to(dev)))
    near(grads[0], gx, E * mp, eps, "grad_x")
    near(grads[1], gg, 2 * E * mp * md, eps, "grad_gate")
    near(grads[2], gi, E * mp, 0.0, "grad_init")
    with torch.no_grad():
        again = gated_ema_forward(*leaves[:2], state_init=leaves[2], lengths=lens, return_state=True)
    assert torch.equal(again[0], h) and torch.equal(again[1], last)
    return h, last, grads


# Within a wave's tokens, a tile, a group of tiles, and past it, forward (16, 128, 1024) and
# backward (8, 64, 512); lane-blocks of 128 channels, odd widths.
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("S", [1, 2, 7, 8, 9, 15, 16, 17, 63, 64, 65, 127, 128, 129, 500, 512, 513, 1023, 1024, 1025, 2500])
def test_lengths_of_sequences(dev, S, dtype):
    check(dev, *make(2, S, 6, dtype, seed=S))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [1, 2, 3, 64, 65, 126, 127, 128, 129, 130, 255, 257, 400])
def test_widths(dev, D, dtype):
    check(dev, *make(3, 150, D, dtype, seed=D))


@pytest.mark.parametrize("B,S,D", [(1, 9000, 3), (40, 140, 20), (9, 700, 130)])
def test_shapes(dev, B, S, D):
    check(dev, *make(B, S, D, seed=1))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_different_lengths(dev, dtype):
    lengths = [700, 0, 1, 64, 65, 128, 129, 699, -3, 900]
    x, gate, init, go, gs = make(10, 700, 33, dtype, seed=2)
    for b, n in enumerate(lengths):      # what is past a row's tokens is not read
        for t in (x, gate, go):
            t[b, max(n, 0):] = float("nan")
    clean = [torch.nan_to_num(t) for t in (x, gate, go)]
    want = reference(clean[0], clean[1], init, clean[2], gs, lengths)
    lens = torch.tensor(lengths, device=dev)
    leaves = [t.to(dev).requires_grad_() for t in (x, gate, init)]
    h, last = gated_ema(*leaves[:2], state_init=leaves[2], lengths=lens, return_state=True)
    grads = torch.autograd.grad((h, last), leaves, (go.to(dev), gs.to(dev)))
    E, eps, (mh, mp, md) = 2.0 ** -24 * (4.0 * (1.0 + 2.0 ** 8.7) + 16.0), EPS[dtype], want[5]   # e^6 < 2^8.7
    for got, ref, bound, e in zip((h.detach(), last.detach(), *grads), want[:5], (E * mh, E * mh, E * mp, 2 * E * mp * md, E * mp),
                                  (eps, 0.0, eps, eps, 0.0)):
        near(got, ref, bound, e, "ragged")
    for b, n in enumerate(lengths):
        for t in (h, grads[0], grads[1]):
            assert (t[b, max(n, 0):] == 0).all()
    assert torch.equal(last[1].detach().cpu(), init[1]) and torch.equal(grads[2][1].cpu(), gs[1])


def test_closed_and_open_gates(dev):
    """Infinite gates: the state stays, or becomes x, exactly; and gates far out."""
    x, gate, init, go, gs = make(2, 300, 5, seed=3)
    gate[:] = float("inf")
    h, last = gated_ema_forward(x.to(dev), gate.to(dev), state_init=init.to(dev), return_state=True)
    assert torch.equal(h.cpu(), init[:, None].expand_as(h)) and torch.equal(last.cpu(), init)
    gate[:] = -float("inf")
    h = gated_ema_forward(x.to(dev), gate.to(dev), state_init=init.to(dev))
    assert torch.equal(h.cpu(), x)
    gate[:, ::2], gate[:, 1::2] = 200.0, -200.0
    check(dev, x, gate.clamp(-80, 25), init, go, gs)
    for g in (float("inf"), -float("inf"), 3e38, -3e38):
        gx, gg, gi = gated_ema_backward(x.to(dev), torch.full_like(gate, g).to(dev), go.to(dev), state_init=init.to(dev),
                                        need_init=True)
        assert (gg == 0).all() and torch.isfinite(gx).all() and torch.isfinite(gi).all()


def test_long_memory_keeps_a_constant(dev):
    """A constant input is a fixed point: decays and weights add up to 1."""
    x = torch.full((1, 20000, 2), 3.0, device=dev)
    gate = torch.full_like(x, 9.0)
    h = gated_ema_forward(x, gate, state_init=torch.full((1, 2), 3.0, device=dev))
    # each step rounds by at most 2^-24 of the state, and the decay pulls back by 1.2e-4 of it
    assert (h - 3.0).abs().max().item() <= 3.0 * 2.0 ** -24 * 2 / 1.2e-4


def test_nan_stays_with_its_channel_and_what_follows(dev):
    x, gate, init, *_ = make(2, 600, 6, seed=4)
    x[0, 300, 2] = float("nan")
    h = gated_ema_forward(x.to(dev), gate.to(dev), state_init=init.to(dev)).cpu()
    assert torch.isnan(h[0, 300:, 2]).all()
    h[0, :, 2] = 0.0
    assert torch.isfinite(h).all()


def test_layouts(dev):
    x, gate, init, go, gs = (t.to(dev) for t in make(3, 200, 96, torch.bfloat16, seed=5))
    want, last = gated_ema_forward(x, gate, state_init=init, return_state=True)
    wide = torch.zeros(3, 200, 203, dtype=x.dtype, device=dev)
    wide[..., 5:101], wide[..., 101:197] = x, gate
    for a, b in ((wide[..., 5:101], wide[..., 101:197]), (x.transpose(0, 1).contiguous().transpose(0, 1), gate),
                 (x, gate.flip(-1).contiguous().flip(-1)), (torch.stack([x, x], -1)[..., 0], gate)):
        assert torch.equal(gated_ema_forward(a, b, state_init=init), want)
    shared = gate[:, :1].expand_as(gate)      # one gate for all tokens: strides of zero
    assert torch.equal(gated_ema_forward(x, shared), gated_ema_forward(x, shared.contiguous()))
    out, state = torch.empty_like(x), init.clone()
    got, fin = gated_ema_forward(x, gate, state_init=state, out=out, state_out=state, return_state=True)
    assert got is out and fin is state and torch.equal(out, want) and torch.equal(state, last)
    full = gated_ema_backward(x, gate, go, state_init=init, grad_state=gs, need_init=True)
    for g in (go.transpose(0, 1).contiguous().transpose(0, 1), torch.stack([go, go], -1)[..., 1]):
        assert all(torch.equal(p, q) for p, q in zip(full, gated_ema_backward(wide[..., 5:101], gate, g, state_init=init,
                                                                              grad_state=gs, need_init=True)))
    one = go[:, :1].expand_as(go)
    assert all(torch.equal(p, q) for p, q in zip(gated_ema_backward(x, gate, one)[:2], gated_ema_backward(x, gate, one.contiguous())[:2]))


def test_states_in_place(dev):
    """The final state where the first was, and the gradients likewise, over several tiles
    and groups of them."""
    for S in (100, 400, 3000):
        x, gate, init, go, gs = (t.to(dev) for t in make(4, S, 384, seed=S))
        want, last = gated_ema_forward(x, gate, state_init=init, return_state=True)
        for _ in range(5):
            state = init.clone()
            got = gated_ema_forward(x, gate, state_init=state, state_out=state)
            assert torch.equal(got, want) and torch.equal(state, last)


def test_types(dev):
    x, gate, init, go, _ = (t.to(dev) for t in make(2, 50, 8, seed=6))
    leaves = x.half().requires_grad_(), gate.bfloat16().requires_grad_(), init.double().requires_grad_()
    h = gated_ema(leaves[0], leaves[1], state_init=leaves[2])
    assert h.dtype == torch.float32
    grads = torch.autograd.grad(h, leaves, go)
    assert [g.dtype for g in grads] == [torch.float16, torch.bfloat16, torch.float64]


def test_pieces_join(dev):
    """A sequence in pieces, the state carried: as the whole."""
    x, gate, init, *_ = make(2, 1000, 40, seed=7)
    out, fin, *_, (mh, _, _) = reference(x, gate, init, torch.zeros_like(x), torch.zeros_like(init))
    E = 2.0 ** -24 * (4.0 * (1.0 + 2.0 ** 8.7) + 16.0)
    state, parts = init.to(dev), []
    for a, b in ((0, 1), (1, 130), (130, 131), (131, 700), (700, 1000)):
        h, state = gated_ema_forward(x[:, a:b].to(dev), gate[:, a:b].to(dev), state_init=state, return_state=True)
        parts.append(h)
    near(torch.cat(parts, 1), out, E * mh, 0.0, "pieces")
    near(state, fin, E * mh, 0.0, "state")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [1, 4, 5, 64, 130, 1030])
def test_step(dev, D, dtype):
    x, gate, init, *_ = make(7, 1, D, dtype, seed=D)
    x, gate = x[:, 0], gate[:, 0]
    want = torch.sigmoid(gate.double()) * init.double() + torch.sigmoid(-gate.double()) * x.double()
    bound, eps = 16 * 2.0 ** -24 * want.abs().max().item() + 2.0 ** -22, EPS[dtype]
    state = init.to(dev)
    near(gated_ema_step(x.to(dev), gate.to(dev), state), want, bound, eps, "out")
    near(state, want, bound, 0.0, "state")
    # scattered slots, one idle row and one past the pool
    pool = torch.full((20, D), 7.0, device=dev)
    slots = torch.tensor([11, 3, -1, 0, 19, 40, 8], device=dev)
    used = [0, 1, 3, 4, 6]
    pool[slots[used]] = init[used].to(dev)
    out = torch.empty(7, D, dtype=dtype, device=dev)
    assert gated_ema_step(x.to(dev), gate.to(dev), pool, slots=slots, out=out) is out
    near(out[used], want[used], bound, eps, "out")
    near(pool[slots[used]], want[used], bound, 0.0, "pool")
    assert (out[2] == 0).all() and torch.isnan(out[5]).all()
    rest = [i for i in range(20) if i not in slots[used].tolist()]
    assert (pool[rest] == 7.0).all()


def test_step_strides_and_alignment(dev):
    x, gate, init, *_ = make(5, 1, 12, seed=8)
    x, gate = x[:, 0].to(dev), gate[:, 0].to(dev)
    state = init.to(dev).clone()
    want = gated_ema_step(x, gate, state)
    wide = torch.zeros(5, 30, device=dev)
    wide[:, 3:15], wide[:, 15:27] = x, gate
    for pool in (torch.zeros(5, 13, device=dev)[:, 1:], torch.zeros(10, 12, device=dev)[::2], torch.zeros(5, 12, device=dev)):
        pool.copy_(init)
        assert torch.equal(gated_ema_step(wide[:, 3:15], wide[:, 15:27], pool), want) and torch.equal(pool, state)


def test_steps_follow_sequences(dev):
    x, gate, init, *_ = make(3, 40, 24, seed=9)
    out, fin, *_, (mh, _, _) = reference(x, gate, init, torch.zeros_like(x), torch.zeros_like(init))
    _, state = gated_ema_forward(x[:, :20].to(dev), gate[:, :20].to(dev), state_init=init.to(dev), return_state=True)
    E = 2.0 ** -24 * (4.0 * (1.0 + 2.0 ** 8.7) + 16.0)
    for t in range(20, 40):
        near(gated_ema_step(x[:, t].to(dev), gate[:, t].to(dev), state), out[:, t], E * mh, 0.0, f"token {t}")
    near(state, fin, E * mh, 0.0, "state")


def test_gradients_against_differences(dev):
    """Central differences of the kernel's forward, h = 2^-7."""
    x, gate, init, go, gs = (t.to(dev) for t in make(2, 90, 7, seed=10, most=3.0))
    leaves = [t.requires_grad_() for t in (x, gate, init)]

    def loss(*t):
        h, last = gated_ema_forward(t[0], t[1], state_init=t[2], return_state=True)
        return (h.double() * go.double()).sum() + (last.double() * gs.double()).sum()

    h, last = gated_ema(*leaves[:2], state_init=leaves[2], return_state=True)
    grads = torch.autograd.grad((h, last), leaves, (go, gs))
    step, gen = 2.0 ** -7, torch.Generator().manual_seed(0)
    for i, grad in enumerate(grads):
        way = torch.randn(grad.shape, generator=gen).to(dev)
        way /= way.norm()
        up, down = (loss(*(t.detach() + s * step * way if j == i else t.detach() for j, t in enumerate(leaves))) for s in (1.0, -1.0))
        got = (grad.double() * way.double()).sum().item()
        # truncation: step^2 of the gradient's size; rounding: 2^-24 of h in 1260 terms over the step
        assert abs((up - down).item() / (2 * step) - got) <= 4 * step * step * grad.norm().item() + 2e-3


def test_only_one_output_is_used(dev):
    x, gate, init, go, gs = (t.to(dev) for t in make(2, 100, 9, seed=11))
    leaves = [t.clone().requires_grad_() for t in (x, gate, init)]

    def grads(*which):
        h, last = gated_ema(*leaves[:2], state_init=leaves[2], return_state=True)
        outs = dict(h=(h, go), s=(last, gs))
        return torch.autograd.grad([outs[w][0] for w in which], leaves, [outs[w][1] for w in which])

    for a, b, c in zip(grads("h", "s"), grads("h"), grads("s")):
        assert (a - b - c).abs().max() <= 1e-4 * (a.abs().max() + b.abs().max() + c.abs().max())
    for i in range(3):
        mine = [t.detach().clone().requires_grad_(j == i) for j, t in enumerate(leaves)]
        gated_ema(*mine[:2], state_init=mine[2]).sum().backward()
        assert [t.grad is not None for t in mine] == [j == i for j in range(3)]


def test_empty(dev):
    init = torch.randn(2, 5, device=dev)
    for B, S in ((2, 0), (0, 3)):
        x = torch.zeros(B, S, 5, device=dev, requires_grad=True)
        i = init[:B].clone().requires_grad_()
        h, last = gated_ema(x, x.detach(), state_init=i, return_state=True)
        gx, gi = torch.autograd.grad((h, last), (x, i), (torch.zeros_like(h), torch.ones_like(last)))
        assert h.shape == (B, S, 5) and torch.equal(last, i) and gx.shape == x.shape and (gi == 1).all()
    h, last = gated_ema_forward(torch.zeros(2, 0, 5, device=dev), torch.zeros(2, 0, 5, device=dev), return_state=True)
    assert (last == 0).all()
    pool = torch.ones(3, 5, device=dev)
    assert gated_ema_step(torch.zeros(0, 5, device=dev), torch.zeros(0, 5, device=dev), pool).shape == (0, 5) and (pool == 1).all()


def test_same_bits_on_every_run_and_graph(dev):
    x, gate, init, go, gs = (t.to(dev) for t in make(3, 3000, 260, torch.bfloat16, seed=12))
    lens = torch.tensor([3000, 1700, 64], dtype=torch.int32, device=dev)
    pool = init.clone()

    def everything():
        h, last = gated_ema_forward(x, gate, state_init=init, lengths=lens, return_state=True)
        pool.copy_(init)
        token = gated_ema_step(x[:, 5], gate[:, 5], pool)
        return (h, last, token, pool.clone(), *gated_ema_backward(x, gate, go, state_init=init, lengths=lens, grad_state=gs,
                                                                  need_init=True))

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
    ins = [[t.to(dev) for t in make(2, 5000, 300, seed=s)] for s in (13, 14)]
    want = [gated_ema_backward(*i[:2], i[3], state_init=i[2]) for i in ins]
    streams = [torch.cuda.Stream(dev) for _ in ins]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for i, s in zip(ins, streams):
            with torch.cuda.stream(s):
                got.append(gated_ema_backward(*i[:2], i[3], state_init=i[2]))
    torch.cuda.synchronize()
    for k, g in enumerate(got):
        assert all(torch.equal(p, q) for p, q in zip(g[:2], want[k % 2][:2]))


def test_refusals(dev):
    x = torch.zeros(2, 6, 8, device=dev)
    state = torch.zeros(3, 8, device=dev)
    for bad in (lambda: gated_ema(x, x[:, :5]), lambda: gated_ema(x[0], x[0]), lambda: gated_ema([1.0], x), lambda: gated_ema(x, None),
                lambda: gated_ema(torch.zeros(2, 3, 0, device=dev), torch.zeros(2, 3, 0, device=dev)),
                lambda: gated_ema(x, x, state_init=state), lambda: gated_ema(x, x, lengths=torch.zeros(2, device=dev)),
                lambda: gated_ema(x, x, lengths=torch.zeros(3, dtype=torch.int32, device=dev)),
                lambda: gated_ema_forward(x, x, out=torch.zeros(2, 6, 9, device=dev)), lambda: gated_ema_forward(x, x.clone(), out=x),
                lambda: gated_ema_forward(x.clone(), x, out=x),
                lambda: gated_ema_forward(x, x, state_out=torch.zeros(2, 9, device=dev)),
                lambda: gated_ema_backward(x, x, x[:1]), lambda: gated_ema_backward(x, x, x, grad_state=state),
                lambda: gated_ema_step(x[0], x[0], state), lambda: gated_ema_step(x[:, 0], x[:, 0], state.bfloat16()),
                lambda: gated_ema_step(x[:, 0], x[:, 0], state[:, :7]), lambda: gated_ema_step(x[:, 0], x[:, 0], state[:1].expand(3, 8)),
                lambda: gated_ema_step(x[:, 0], x[:, 0], state, slots=torch.zeros(2, dtype=torch.int32, device=dev)),
                lambda: gated_ema_step(x[:, 0], x[:, 0], state, slots=torch.zeros(3, dtype=torch.int64, device=dev)),
                lambda: gated_ema_step(x[:, 0], x[:, 0], state, out=state[:2])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="ROCm GPU only"):
        gated_ema(x.cpu(), x.cpu())
