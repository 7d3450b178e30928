"""The gated EMA, the residual norm and the vocabulary's cross entropy through the
extension module and through ctypes: the same bits, the same graph, the same
refusals; and a training step that runs them together."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from orthossm_amd import _native as nat
from orthossm_amd import (block_norm, clip_grad_norm, ema, gated_ema, gated_ema_forward, gated_ema_step, linear_cross_entropy,
                          linear_loss, ops, residual_norm)

pytestmark = pytest.mark.gpu


def through_ctypes(monkeypatch):
    for module in (ema, block_norm, linear_loss):
        monkeypatch.setattr(module, "_fast", lambda: None)


@pytest.fixture(params=["extension", "ctypes"])
def path(request, monkeypatch):
    if request.param == "ctypes":
        through_ctypes(monkeypatch)
    else:
        assert ops._fast() is not None
    return request.param


def rand(*shape, seed, dtype=torch.float32, dev="cuda"):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(dev)


def ema_inputs(dtype=torch.float32, S=150):
    return [rand(2, S, 24, seed=1, dtype=dtype), 2 + rand(2, S, 24, seed=2, dtype=dtype), rand(2, 24, seed=3)]


def block_inputs(dtype=torch.float32):
    return [rand(4, 40, seed=4), *(rand(4, 40, seed=s, dtype=dtype) for s in (5, 6)), *(rand(40, seed=s) for s in (7, 8, 9))]


def loss_inputs(dtype=torch.float32):
    return [rand(20, 32, seed=10, dtype=dtype), rand(50, 32, seed=11, dtype=dtype)]


def targets():
    t = torch.arange(20, device="cuda") * 2
    t[3] = -100
    return t


# name: (leaves, call), the call giving one or more outputs
CALLS = {
    "ema": (ema_inputs, lambda t: gated_ema(t[0], t[1], state_init=t[2], return_state=True)),
    "ema ragged": (ema_inputs, lambda t: gated_ema(t[0], t[1], state_init=t[2], return_state=True,
                                                   lengths=torch.tensor([150, 33], dtype=torch.int32, device="cuda"))),
    "block": (block_inputs, lambda t: residual_norm(t[0], t[1], t[4], t[5], gate=t[2], scale=t[3])),
    "block rms": (block_inputs, lambda t: residual_norm(t[0], t[1], t[4], gate=t[2], scale=t[3], rms=True, norm_y=False)),
    "loss": (loss_inputs, lambda t: (linear_cross_entropy(t[0], t[1], targets()),)),
    "loss sum": (loss_inputs, lambda t: (linear_cross_entropy(t[0], t[1], targets(), reduction="sum"),)),
    "loss none": (loss_inputs, lambda t: (linear_cross_entropy(t[0], t[1], targets(), reduction="none"),)),
}


def run(name, dtype=torch.float32):
    make, call = CALLS[name]
    leaves = [t.requires_grad_() for t in make(dtype)]
    outs = call(leaves)
    grads = torch.autograd.grad(outs, leaves, [0.5 * torch.ones_like(o) for o in outs], allow_unused=True)
    return [*outs, *(g for g in grads if g is not None)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", CALLS)
def test_both_paths_give_the_same_bits(dev, name, dtype, monkeypatch):
    def calls():
        res = run(name, dtype)
        with torch.no_grad():
            res += CALLS[name][1](CALLS[name][0](dtype))
        return res

    assert ops._fast() is not None
    want = calls()
    through_ctypes(monkeypatch)
    got = calls()
    assert len(want) == len(got)
    for a, b in zip(want, got):
        assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b)


def test_steps_give_the_same_bits(dev, monkeypatch):
    x, gate, state = ema_inputs()
    slots = torch.tensor([1, 0], device=dev)

    def step():
        pool = state.clone()
        return gated_ema_step(x[:, 0], gate[:, 1], pool, slots=slots), pool

    want = step()
    through_ctypes(monkeypatch)
    assert all(torch.equal(a, b) for a, b in zip(want, step()))


@pytest.mark.parametrize("name", CALLS)
def test_only_what_requires_a_gradient_gets_one(dev, path, name):
    make, call = CALLS[name]
    for i in range(len(make())):
        leaves = [t.requires_grad_(j == i) for j, t in enumerate(make())]
        outs = call(leaves)
        if name == "block rms" and i == 5:      # (no bias in this form)
            assert not any(o.requires_grad for o in outs)
            continue
        assert all(o.requires_grad for o in outs)
        sum(o.sum() for o in outs).backward()      # (broadcast gradients: strides of zero)
        assert [t.grad is not None for t in leaves] == [j == i for j in range(len(leaves))]
    with torch.no_grad():
        assert not any(o.requires_grad for o in call([t.requires_grad_() for t in make()]))


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", CALLS)
def test_forward_mode_is_refused(dev, path, name, grad):
    make, call = CALLS[name]
    with forward_ad.dual_level():
        for i in range(5 if name.startswith("block") else len(make())):
            mine = [t.requires_grad_(grad) for t in make()]
            mine[i] = forward_ad.make_dual(mine[i], torch.ones_like(mine[i]))
            with pytest.raises(NotImplementedError, match="forward mode"):
                call(mine)
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward mode"):
                call(mine)


@pytest.mark.parametrize("name", CALLS)
def test_gradients_can_be_differentiated_once_only(dev, path, name):
    make, call = CALLS[name]
    leaves = [t.requires_grad_() for t in make()]
    outs = call(leaves)
    grads = torch.autograd.grad(sum((o * o).sum() for o in outs), leaves, create_graph=True, allow_unused=True)
    with pytest.raises(RuntimeError, match="twice"):
        sum(t.sum() for t in grads if t is not None).backward()


@pytest.mark.parametrize("name", CALLS)
def test_a_changed_input_is_refused_in_the_backward(dev, path, name):
    make, call = CALLS[name]
    for i in range(2):
        leaves = [t.requires_grad_() for t in make()]
        outs = call(leaves)
        with torch.no_grad():
            leaves[i].mul_(2)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            sum(o.sum() for o in outs).backward()


@pytest.mark.parametrize("name", CALLS)
def test_a_changed_output_does_not_matter(dev, path, name):
    """Nothing that the backward reads is handed out."""
    make, call = CALLS[name]
    leaves = [t.requires_grad_() for t in make()]
    want = run(name)
    outs = call(leaves)
    ones = [0.5 * torch.ones_like(o) for o in outs]
    with torch.no_grad():
        for o in outs:
            o.detach().zero_()
    grads = [g for g in torch.autograd.grad(outs, leaves, ones, allow_unused=True) if g is not None]
    assert all(torch.equal(a, b) for a, b in zip(want[len(outs):], grads))


@pytest.mark.parametrize("name", CALLS)
def test_saved_tensor_hooks(dev, path, name):
    want = run(name)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), lambda t: t.clone()):
        got = run(name)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("name", CALLS)
def test_saved_tensors_of_another_form_are_refused(dev, path, name):
    """A hook may give back anything: what does not fit is not read."""
    make, call = CALLS[name]
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append(t.shape) or t, lambda t: t):
        call([t.requires_grad_() for t in make()])
    for k in range(len(seen)):
        if len(seen[k]) == 0 or seen[k].numel() < 2:
            continue
        count = iter(range(len(seen) + 9))
        with torch.autograd.graph.saved_tensors_hooks(lambda t: (next(count), t), lambda p: p[1][: p[1].shape[0] // 2] if p[0] == k else p[1]):
            outs = call([t.requires_grad_() for t in make()])
        with pytest.raises((RuntimeError, ValueError)):
            sum(o.sum() for o in outs).backward()


def test_writes_are_seen_by_graphs_that_saved_the_tensor(dev, path):
    x, gate, state = ema_inputs()
    out, h, last = torch.zeros(2, 24, device=dev), torch.zeros(2, 150, 24, device=dev), state.clone()
    for t, call in ((state, lambda: gated_ema_step(x[:, 0], gate[:, 0], state)),
                    (out, lambda: gated_ema_step(x[:, 0], gate[:, 0], state.clone(), out=out)),
                    (h, lambda: gated_ema_forward(x, gate, out=h)),
                    (last, lambda: gated_ema_forward(x, gate, state_init=last, return_state=True, state_out=last))):
        factor = torch.ones_like(t, requires_grad=True)
        product = t * factor
        call()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            product.sum().backward()
    with torch.inference_mode():
        pool = state.clone()
        gated_ema_step(x[:, 0], gate[:, 0], pool)
    before = pool.clone()
    gated_ema_step(x[:, 0], gate[:, 0], pool)
    assert not torch.equal(pool, before)
    leaf = torch.zeros(2, 24, device=dev, requires_grad=True)
    with pytest.raises(ValueError, match="gradient"):
        gated_ema_step(x[:, 0], gate[:, 0], state, out=leaf)
    with pytest.raises(ValueError):
        gated_ema_step(x[:, 0], gate[:, 0], leaf)


def test_outputs_in_an_arguments_memory(dev, path):
    x, gate, state = ema_inputs()
    store = torch.zeros(3, 24, device=dev)
    for call in (lambda: gated_ema_forward(x, gate, out=x), lambda: gated_ema_forward(x, gate, out=gate),
                 lambda: gated_ema_forward(x, gate, state_out=x.view(-1)[:48].view(2, 24)),
                 lambda: gated_ema_step(store[:2], gate[:, 0], state, out=store[1:]),
                 lambda: gated_ema_step(x[:, 0], gate[:, 0], store, out=store[1:])):
        with pytest.raises(ValueError, match="shares memory"):
            call()


def test_errors_of_the_library(dev, path):
    with pytest.raises(nat.OsmError):
        residual_norm(*block_inputs()[:2], eps=-1.0)
    with pytest.raises(nat.OsmError):
        linear_cross_entropy(torch.zeros(2, 1 << 18, device=dev), torch.zeros(1, 1 << 18, device=dev),
                             torch.zeros(2, dtype=torch.int64, device=dev))


@pytest.mark.parametrize("name", CALLS)
def test_on_another_stream(dev, path, name):
    want = run(name)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = run(name)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("name", ["ema", "block", "block rms", "loss", "loss sum", "loss none"])
def test_a_captured_training_pass(dev, path, name, monkeypatch):
    """Forward and backward in a graph, replayed between eager passes over the same leaves
    (none of which is alive while the graph is captured)."""
    make, call = CALLS[name]
    goal = targets()
    monkeypatch.setitem(globals(), "targets", lambda: goal)   # (made from the host)
    leaves = [t.requires_grad_() for t in make()]
    weights = [torch.full_like(o, 0.5) for o in call([t.detach() for t in leaves])]

    def once():
        outs = call(leaves)
        grads = torch.autograd.grad(outs, leaves, weights, allow_unused=True)
        return [o.detach() for o in outs] + [g for g in grads if g is not None]

    want = [t.clone() for t in once()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = once()
    for _ in range(3):
        for t in held:
            t.zero_()
        graph.replay()
        got = once()
        torch.cuda.synchronize()
        for a, b, c in zip(want, got, held):
            assert torch.equal(a, b) and torch.equal(a, c)


class Model(torch.nn.Module):
    """Layers of the gated EMA between residual norms, and the loss."""

    def __init__(self, vocabulary, width, layers):
        super().__init__()
        gen = torch.Generator().manual_seed(0)

        def p(*shape, scale=1.0, base=0.0):
            return torch.nn.Parameter(base + scale * torch.randn(*shape, generator=gen))

        self.table, self.first = p(vocabulary, width, scale=0.5), p(width, scale=0.1, base=1.0)
        self.layers = torch.nn.ModuleList()
        for _ in range(layers):
            m = torch.nn.Module()
            m.win, m.wout = p(width, 3 * width, scale=width ** -0.5), p(width, width, scale=width ** -0.5)
            m.scale, m.weight, m.bias = p(width, scale=0.1, base=0.5), p(width, scale=0.1, base=1.0), p(width, scale=0.1)
            self.layers.append(m)

    def forward(self, tokens, lengths, block, recur, norm):
        r = self.table[tokens]
        n = norm(r, self.first)
        for m in self.layers:
            x, f, g = (n @ m.win).split(n.shape[-1], -1)
            r, n = block(r, recur(x, f + 2, lengths) @ m.wout, m.weight, m.bias, g, m.scale)
        return n


def test_a_training_step_and_serving(dev, path):
    """A model of these operators: its loss and gradients against the same model in
    float64, clipped; then its prompt read whole and answered token by token."""
    V, D, B, S = 300, 48, 3, 200
    model = Model(V, D, 2).to(dev)
    tokens = torch.randint(V, (B, S), generator=torch.Generator().manual_seed(1)).to(dev)
    lengths = torch.tensor([200, 77, 129], dtype=torch.int32, device=dev)
    goal = torch.roll(tokens, -1, 1)
    goal[torch.arange(S, device=dev)[None, :] >= lengths[:, None]] = -100

    def norm(v, w, b=0.0):
        v = v - v.mean(-1, keepdim=True)
        return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-5) * w + b

    def plain_ema(x, f, lens):
        a, h, out = torch.sigmoid(f), torch.zeros_like(x[:, 0]), []
        for t in range(x.shape[1]):
            h = a[:, t] * h + (1 - a[:, t]) * x[:, t]
            out.append(h)
        used = torch.arange(x.shape[1], device=x.device)[None, :] < lens[:, None]
        return torch.where(used[..., None], torch.stack(out, 1), 0.0)

    def plain_block(r, y, w, b, g, s):
        r = r + s * torch.sigmoid(g) * norm(y, 1.0)
        return r, norm(r, w, b)

    def own_block(r, y, w, b, g, s):
        return residual_norm(r, y, w, b, gate=g, scale=s)

    def own_ema(x, f, lens):
        return gated_ema(x, f, lengths=lens)

    n = model(tokens, lengths, own_block, own_ema, norm)
    loss = linear_cross_entropy(n, model.table, goal)
    loss.backward()
    twin = Model(V, D, 2).double().to(dev)
    nd = twin(tokens, lengths, plain_block, plain_ema, norm)
    want = torch.nn.functional.cross_entropy((nd @ twin.table.t()).flatten(0, 1), goal.flatten())
    want.backward()
    assert abs(loss.item() - want.item()) <= 1e-5 * want.item()
    total = sum(p.grad.square().sum() for p in twin.parameters()).sqrt()
    for p, q in zip(model.parameters(), twin.parameters()):
        # torch's fp32 products over 48 to 600 terms and five layers of norms between: 1e-4 of the gradient's size
        assert (p.grad - q.grad).norm() <= 1e-4 * q.grad.norm() + 1e-6 * total
    got = clip_grad_norm([p.grad for p in model.parameters()], 1.0)
    assert abs(got.item() - total.item()) <= 1e-4 * total.item()

    # serving: the states after the prompts move into a pool, in another order
    with torch.no_grad():
        slots = torch.tensor([4, 0, 3], device=dev)
        pools = [torch.zeros(5, D, device=dev) for _ in model.layers]
        which = iter(pools)

        def prompt_ema(x, f, lens):
            h, state = gated_ema(x, f, lengths=lens, return_state=True)
            next(which)[slots] = state
            return h

        model(tokens, torch.tensor([150, 76, 100], device=dev), own_block, prompt_ema, norm)
        for step in range(3):
            at = torch.tensor([150, 76, 100], device=dev) + step
            live = at < lengths
            which = iter(pools)

            def token_ema(x, f, lens):
                return gated_ema_step(x, f, next(which), slots=torch.where(live, slots, -1))

            one = model(tokens[torch.arange(B, device=dev), at], None, own_block, token_ema, norm)
            rows = n[torch.arange(B, device=dev), at][live]
            assert (one[live] - rows).abs().max() <= 1e-4 * rows.abs().max()
