"""The gated delta rule, the layer norm and the clipping through the extension
module and through ctypes: the same bits, the same graph, the same refusals."""
import pytest
import torch

from orthossm_amd import _native as nat
from orthossm_amd import clip_grad_norm, delta, gated_delta, gated_delta_step, grad_clip, grad_norm, layer_norm, norm, ops

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["extension", "ctypes"])
def path(request, monkeypatch):
    if request.param == "ctypes":
        for module in (delta, norm, grad_clip):
            monkeypatch.setattr(module, "_fast", lambda: None)
    else:
        assert ops._fast() is not None
    return request.param


def delta_inputs(dev, dtype=torch.float32, B=2, S=70, H=4, Hk=2, dk=24, dv=20):
    gen = torch.Generator().manual_seed(5)
    q, k = (torch.nn.functional.normalize(torch.randn(B, S, Hk, dk, generator=gen), dim=-1).to(dtype) for _ in range(2))
    v = torch.randn(B, S, H, dv, generator=gen).to(dtype)
    g, beta = -torch.rand(B, S, H, generator=gen), torch.rand(B, S, H, generator=gen)
    init = torch.randn(B, H, dk, dv, generator=gen)
    return [t.to(dev).requires_grad_() for t in (q, k, v, g, beta, init)]


def delta_pass(ins, lengths):
    out, fin = gated_delta(*ins[:5], state_init=ins[5], lengths=lengths, return_state=True)
    return out, fin, *torch.autograd.grad((out, fin), ins, (torch.ones_like(out), torch.ones_like(fin)))


def norm_inputs(dev, dtype=torch.float32):
    gen = torch.Generator().manual_seed(6)
    return [t.to(dev).requires_grad_() for t in (torch.randn(3, 50, 40, generator=gen).to(dtype),
                                                 torch.randn(40, generator=gen), torch.randn(40, generator=gen))]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_both_paths_give_the_same_bits(dev, dtype, monkeypatch):
    ins, lengths = delta_inputs(dev, dtype), torch.tensor([70, 33], dtype=torch.int32, device=dev)
    x = norm_inputs(dev, dtype)
    token = [t.detach()[:, 0].contiguous() for t in ins[:5]]
    grads = [t.detach().clone() for t in ins]

    def calls():
        res = list(delta_pass(ins, lengths))
        y = layer_norm(*x)
        res += [y, *torch.autograd.grad(y, x, y.detach())]
        with torch.no_grad():
            res += [*gated_delta(*ins[:5], lengths=lengths, return_state=True), layer_norm(*x)]
        state = ins[5].detach().clone()
        res += [gated_delta_step(*token, state), state]
        clipped = [t.clone() for t in grads]
        res += [grad_norm(grads), clip_grad_norm(clipped, 0.5), *clipped]
        return res

    assert ops._fast() is not None
    want = calls()
    for module in (delta, norm, grad_clip):
        monkeypatch.setattr(module, "_fast", lambda: None)
    got = calls()
    assert len(want) == len(got)
    for a, b in zip(want, got):
        assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b)


def test_only_what_requires_a_gradient_gets_one(dev, path):
    ins = [t.detach() for t in delta_inputs(dev)]
    for i in range(6):
        mine = [t.clone().requires_grad_(j == i) for j, t in enumerate(ins)]
        out, fin = gated_delta(*mine[:5], state_init=mine[5], return_state=True)
        assert out.requires_grad and fin.requires_grad
        (out.sum() + fin.sum()).backward()       # (a broadcast gradient: strides of zero)
        assert [t.grad is not None for t in mine] == [j == i for j in range(6)]
    x = [t.detach() for t in norm_inputs(dev)]
    for i in range(3):
        mine = [t.clone().requires_grad_(j == i) for j, t in enumerate(x)]
        layer_norm(*mine).sum().backward()
        assert [t.grad is not None for t in mine] == [j == i for j in range(3)]
    with torch.no_grad():
        assert not layer_norm(*norm_inputs(dev)).requires_grad
        assert not gated_delta(*delta_inputs(dev)[:5]).requires_grad


def test_absent_and_unused(dev, path):
    ins = delta_inputs(dev)
    whole = delta_pass(ins, None)
    out, fin = gated_delta(*ins[:5], state_init=ins[5], return_state=True)
    from_out = torch.autograd.grad(out, ins, torch.ones_like(out))
    out, fin = gated_delta(*ins[:5], state_init=ins[5], return_state=True)
    from_state = torch.autograd.grad(fin, ins, torch.ones_like(fin), allow_unused=True)
    for a, b, c in zip(whole[2:], from_out, from_state):
        # sums of up to 70 tokens' terms in another order
        assert (a - b - c).abs().max() <= 1e-4 * (a.abs().max() + b.abs().max() + c.abs().max())
    assert gated_delta(*ins[:5]).requires_grad      # no first state, no final one
    x, w, _ = norm_inputs(dev)
    for weight in (None, w):
        gx, = torch.autograd.grad(layer_norm(x, weight), x, torch.ones_like(x))
        assert gx.shape == x.shape


def test_gradients_can_be_differentiated_once_only(dev, path):
    for ins, make in ((delta_inputs(dev), lambda t: gated_delta(*t[:5], state_init=t[5])),
                      (norm_inputs(dev), lambda t: layer_norm(*t))):
        out = make(ins)
        grads = torch.autograd.grad((out * out).sum(), ins, create_graph=True)
        assert all(t.requires_grad for t in grads)
        with pytest.raises(RuntimeError, match="twice"):
            sum(t.sum() for t in grads).backward()


def test_a_changed_input_is_refused_in_the_backward(dev, path):
    x, w, b = norm_inputs(dev)
    y = layer_norm(x, w, b)
    with torch.no_grad():
        x.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_saved_tensor_hooks(dev, path):
    ins, x = delta_inputs(dev), norm_inputs(dev)
    want = delta_pass(ins, None)
    y = layer_norm(*x)
    want_norm = torch.autograd.grad(y, x, torch.ones_like(y))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), lambda t: t.clone()):
        got = delta_pass(ins, None)
        y = layer_norm(*x)
    for a, b in zip((*want, *want_norm), (*got, *torch.autograd.grad(y, x, torch.ones_like(y)))):
        assert torch.equal(a, b)


def test_errors_of_the_library(dev, path):
    with pytest.raises(nat.OsmError):
        layer_norm(norm_inputs(dev)[0], eps=-1.0)


def test_on_another_stream(dev, path):
    ins = delta_inputs(dev)
    want = delta_pass(ins, None)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = delta_pass(ins, None)
    side.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)
