"""What torch's autograd has to see of the gated delta rule, the layer norm and
the clipping, through the extension module and through ctypes."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from orthossm_amd import (clip_grad_norm, delta, gated_delta, gated_delta_forward, gated_delta_step, grad_clip, grad_norm,
                          layer_norm, layer_norm_forward, norm, ops)

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["extension", "ctypes"])
def path(request, monkeypatch):
    if request.param == "ctypes":
        for module in (delta, norm, grad_clip):
            monkeypatch.setattr(module, "_fast", lambda: None)
    else:
        assert ops._fast() is not None
    return request.param


def delta_inputs(dev, S=20):
    gen = torch.Generator().manual_seed(2)
    shapes = ((2, S, 1, 8), (2, S, 1, 8), (2, S, 2, 12), (2, S, 2), (2, S, 2), (2, 2, 8, 12))
    t = [0.3 * torch.randn(s, generator=gen) for s in shapes]
    return [x.to(dev) for x in (*t[:3], -t[3].abs(), *t[4:])]


def norm_inputs(dev):
    gen = torch.Generator().manual_seed(3)
    return [torch.randn(s, generator=gen).to(dev) for s in ((4, 40), (40,), (40,))]


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(dev, path, grad):
    """No forward-mode derivative exists: an error, not a derivative of zero."""
    with forward_ad.dual_level():
        for ins, call in ((delta_inputs(dev), lambda t: gated_delta(*t[:5], state_init=t[5])),
                          (norm_inputs(dev), lambda t: layer_norm(*t))):
            for i in range(len(ins)):
                mine = [t.clone().requires_grad_(grad) for t in ins]
                mine[i] = forward_ad.make_dual(mine[i], torch.ones_like(ins[i]))
                with pytest.raises(NotImplementedError, match="forward mode"):
                    call(mine)
                with torch.no_grad(), pytest.raises(NotImplementedError, match="forward mode"):
                    call(mine)


def token(dev):
    return [t[:, 0].contiguous() for t in delta_inputs(dev)[:5]]


def writers(dev):
    """name: (the tensor a call writes into, the call)."""
    ins, (x, w, b) = delta_inputs(dev), norm_inputs(dev)
    state, out, first = ins[5].clone(), torch.zeros(2, 2, 12, device=dev), torch.zeros(2, 20, 2, 12, device=dev)
    last, y = ins[5].clone(), x.clone()
    grads = [torch.ones(9, device=dev), torch.ones(20, 6, device=dev)[:, ::2]]
    return {
        "step's state": (state, lambda: gated_delta_step(*token(dev), state)),
        "step's out": (out, lambda: gated_delta_step(*token(dev), ins[5].clone(), out=out)),
        "out": (first, lambda: gated_delta_forward(*ins[:5], out=first)),
        "state_out": (last, lambda: gated_delta_forward(*ins[:5], state_init=last, return_state=True, state_out=last)),
        "norm's out": (y, lambda: layer_norm_forward(y, w, b, out=y)),
        "a gradient": (grads[0], lambda: clip_grad_norm(grads, 1.0)),
        "a gradient with gaps": (grads[1], lambda: clip_grad_norm(grads, 1.0)),
    }


WRITERS = ["step's state", "step's out", "out", "state_out", "norm's out", "a gradient", "a gradient with gaps"]


@pytest.mark.parametrize("name", WRITERS)
def test_writes_are_seen_by_graphs_that_saved_the_tensor(dev, path, name):
    t, call = writers(dev)[name]
    factor = torch.ones_like(t, requires_grad=True)
    for _ in range(2):      # the second time after a write of the first
        product = t * factor
        (product.sum()).backward()
        product = t * factor
        call()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            product.sum().backward()


def test_reads_are_not_writes(dev, path):
    ins, (x, w, b) = delta_inputs(dev), norm_inputs(dev)
    ts = [*ins, x, w, b]
    before = [t._version for t in ts]
    gated_delta_forward(*ins[:5], state_init=ins[5], return_state=True)
    layer_norm_forward(x, w, b)
    grad_norm(ts)
    assert [t._version for t in ts] == before


@pytest.mark.parametrize("name", WRITERS)
def test_inference_tensors_are_written(dev, path, name):
    with torch.inference_mode():
        t, call = writers(dev)[name]
        before = t.clone()
        call()
    assert not torch.equal(t, before)


def test_a_pool_made_in_inference_mode_serves_outside_it(dev, path):
    with torch.inference_mode():
        state = delta_inputs(dev)[5].clone()
    before = state.clone()
    gated_delta_step(*token(dev), state)
    assert not torch.equal(state, before)


def test_outputs_that_require_a_gradient_are_refused(dev, path):
    ins, (x, w, b) = delta_inputs(dev), norm_inputs(dev)

    def leaf(*shape):
        return torch.zeros(*shape, device=dev, requires_grad=True)

    calls = (lambda: gated_delta_forward(*ins[:5], out=leaf(2, 20, 2, 12)),
             lambda: gated_delta_forward(*ins[:5], return_state=True, state_out=leaf(2, 2, 8, 12)),
             lambda: gated_delta_step(*token(dev), ins[5].clone(), out=leaf(2, 2, 12)),
             lambda: layer_norm_forward(x, w, b, out=leaf(4, 40)))
    for call in calls:
        with pytest.raises(ValueError, match="gradient"):
            call()
        with torch.no_grad():
            call()


def half_of(is_one):
    """Hooks that give back half of the saved tensors that ``is_one`` picks."""
    return torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t[:t.shape[0] // 2] if is_one(t) else t)


@pytest.mark.parametrize("which", ["what the forward kept", "lengths", "statistics", "weight", "input"])
def test_saved_tensors_of_another_form_are_refused(dev, path, which):
    """A hook may give back anything: what does not fit is not read."""
    lengths = torch.tensor([20, 7], dtype=torch.int32, device=dev)
    picks = {"what the forward kept": lambda t: t.dtype == torch.uint8, "lengths": lambda t: t.dtype == torch.int32,
             "statistics": lambda t: t.shape == (4,), "weight": lambda t: t.shape == (40,),
             "input": lambda t: t.shape in ((2, 20, 2, 12), (4, 40))}
    ins = [t.requires_grad_() for t in delta_inputs(dev)]
    x = [t.requires_grad_() for t in norm_inputs(dev)]
    with half_of(picks[which]):
        outs = []
        if which not in ("statistics", "weight"):
            outs.append(gated_delta(*ins[:5], state_init=ins[5], lengths=lengths))
        if which not in ("what the forward kept", "lengths"):
            outs.append(layer_norm(*x))
    for out in outs:
        with pytest.raises((RuntimeError, ValueError)):
            out.sum().backward()


def test_outputs_in_an_arguments_memory(dev, path):
    """out may be v, the norm's x, state_out the first state; nothing else."""
    gen = torch.Generator().manual_seed(4)
    q, k, v = (torch.randn(2, 70, 2, 16, generator=gen).to(dev) for _ in range(3))
    g, beta, init = -torch.ones(2, 70, 2, device=dev), torch.full((2, 70, 2), 0.5, device=dev), torch.ones(2, 2, 16, 16, device=dev)
    want, fin = gated_delta_forward(q, k, v, g, beta, state_init=init, return_state=True)
    last, mine = init.clone(), v.clone()
    gated_delta_forward(q, k, mine, g, beta, state_init=last, out=mine, return_state=True, state_out=last)
    assert torch.equal(mine, want) and torch.equal(last, fin)
    one = [t[:, 0].contiguous() for t in (q, k, v, g, beta)]
    state, want = init.clone(), gated_delta_step(*one, init.clone())
    assert torch.equal(gated_delta_step(*one, state, out=one[2]), want)
    one[2] = v[:, 0].contiguous()
    x, w, b = norm_inputs(dev)
    store = torch.zeros(5, 40, device=dev)
    for call in (lambda: gated_delta_forward(q, k, v, g, beta, out=q), lambda: gated_delta_forward(q, k, v, g, beta, out=k),
                 lambda: gated_delta_forward(q, k, v, g, beta, state_out=q.view(-1)[:1024].view(2, 2, 16, 16)),
                 lambda: gated_delta_step(*one, state, out=one[0]),
                 lambda: gated_delta_step(*one, state, out=state.view(-1)[64:128].view(2, 2, 16)),
                 lambda: layer_norm_forward(store[:4], w, b, out=store[1:]),
                 lambda: layer_norm_forward(store[:1], store[1], b, out=store[1:2])):
        with pytest.raises(ValueError, match="shares memory"):
            call()
