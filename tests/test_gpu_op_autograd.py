"""What torch's autograd has to see of the gated delta rule, the layer norm and
the clipping, through the extension module and through ctypes."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from orthossm_amd import delta, gated_delta, grad_clip, layer_norm, norm, ops

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
