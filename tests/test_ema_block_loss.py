"""CPU checks of the gated EMA's, the residual norm's and the vocabulary's cross
entropy's C entry points: sizes and refusals, which come back as status codes
before any HIP call."""
import ctypes

import pytest
import torch

from orthossm_amd import _native as nat
from orthossm_amd import gated_ema, gated_ema_step, linear_cross_entropy, residual_norm

P = 0x10000      # never dereferenced: every case is refused


@pytest.fixture(autouse=True)
def _no_message_left():
    """A call that succeeds clears the thread's message."""
    yield
    a = nat.NormArgs()
    a.abi_version, a.D = nat.ABI_VERSION, 1
    assert nat.load().osm_layer_norm_fwd(ctypes.byref(a), None) == 0


def made(cls, **kw):
    a = cls()
    a.abi_version = nat.ABI_VERSION
    for k, v in kw.items():
        if "." in k:
            part, field = k.split(".")
            setattr(getattr(a, part), field, v)
        else:
            setattr(a, k, v)
    return a


def seqs(*names, S=300, D=40):
    return {f"{n}.{f}": v for n in names for f, v in (("p", P), ("stride_b", S * D), ("stride_s", D))}


def ema(**kw):
    return made(nat.EmaArgs, **{**dict(B=2, S=300, D=40, saved=P), **seqs("x", "gate", "out"), **kw})


def test_ema_sizes():
    lib = nat.load()
    # maps of 3 tiles of 128 channels, one group's state, a counter on a line of its own; backward 5 tiles
    for f, tiles in ((lib.osm_gated_ema_workspace_bytes, 3), (lib.osm_gated_ema_bwd_workspace_bytes, 5)):
        assert f(ctypes.byref(ema())) == 2 * (tiles * 128 * 8 + 128 * 8 + 128)
        assert f(ctypes.byref(ema(S=64))) == f(ctypes.byref(ema(B=0))) == f(ctypes.byref(ema(S=0))) == 0
        assert f(ctypes.byref(ema(D=0))) == 0
    assert lib.osm_gated_ema_workspace_bytes(ctypes.byref(ema(S=128))) == 0
    assert lib.osm_gated_ema_saved_bytes(ctypes.byref(ema())) == 2 * 5 * 40 * 4


COMMON = [(dict(abi_version=1), -1), (dict(dtype=2), -3)]
EMA_ERRORS = COMMON + [(dict(B=-1), -2), (dict(D=0), -2), (dict(S=-1), -2), (dict(S=1 << 31), -2), (dict(B=1 << 31), -2),
                       (dict(B=1 << 20, D=4096), -2), ({"x.p": None}, -1), ({"gate.p": P + 2}, -4), ({"x.stride_s": -40}, -4),
                       ({"gate.stride_b": -1}, -4), (dict(lengths=P + 2), -4), (dict(state_init=P + 1), -4), (dict(saved=P + 2), -4)]


@pytest.mark.parametrize("kw,code", EMA_ERRORS + [({"out.p": None}, -1), ({"out.stride_s": 39}, -4), ({"out.stride_b": 40}, -4),
                                                  ({"out.stride_b": 0}, -4)])
def test_ema_errors(kw, code):
    lib = nat.load()
    assert lib.osm_gated_ema_fwd(ctypes.byref(ema(**kw)), ctypes.c_void_p(P), 1 << 40, None) == code
    assert lib.osm_last_error() != b""


@pytest.mark.parametrize("kw,bwd,code", [(kw, {}, code) for kw, code in EMA_ERRORS] + [
    (dict(saved=None), {}, -1), ({}, {"grad_out.p": None}, -1), ({}, {"grad_x.stride_s": 20}, -4), ({}, {"grad_gate.p": P + 1}, -4),
    ({}, {"grad_out.stride_s": -40}, -4), ({}, dict(grad_state=P + 2), -4), ({}, dict(grad_init=P + 2), -4)])
def test_ema_backward_errors(kw, bwd, code):
    b = made(nat.EmaBwdArgs, **{**seqs("grad_out", "grad_x", "grad_gate"), **bwd})
    assert nat.load().osm_gated_ema_bwd(ctypes.byref(ema(**kw)), ctypes.byref(b), ctypes.c_void_p(P), 1 << 40, None) == code


def test_ema_workspace_errors():
    lib, b = nat.load(), made(nat.EmaBwdArgs, **seqs("grad_out", "grad_x", "grad_gate"))
    need = lib.osm_gated_ema_workspace_bytes(ctypes.byref(ema())), lib.osm_gated_ema_bwd_workspace_bytes(ctypes.byref(ema()))
    for ws, less in ((None, 0), (P + 16, 0), (P, 1)):
        assert lib.osm_gated_ema_fwd(ctypes.byref(ema()), ctypes.c_void_p(ws), need[0] - less, None) == -5
        assert lib.osm_gated_ema_bwd(ctypes.byref(ema()), ctypes.byref(b), ctypes.c_void_p(ws), need[1] - less, None) == -5
    assert lib.osm_gated_ema_bwd(ctypes.byref(ema()), None, ctypes.c_void_p(P), 1 << 40, None) == -1
    assert lib.osm_gated_ema_fwd(None, None, 0, None) == -1 and lib.osm_gated_ema_step(None, None) == -1


@pytest.mark.parametrize("kw,code", COMMON + [
    (dict(B=-1), -2), (dict(D=0), -2), (dict(n_slots=3), -2), (dict(n_slots=-1, slots=P), -2), ({"x.p": None}, -1), ({"gate.p": P + 1}, -4),
    ({"out.stride_b": 39}, -4), (dict(state=None), -1), (dict(state=P + 2), -4), (dict(slots=P + 4), -4), (dict(state_stride=39), -4),
    (dict(B=1 << 20, D=1 << 13, n_slots=1 << 20), -2)])
def test_ema_step_errors(kw, code):
    a = made(nat.EmaStepArgs, **{**dict(B=4, D=40, state=P, state_stride=40, n_slots=4),
                                 **{f"{n}.{f}": v for n in ("x", "gate", "out") for f, v in (("p", P), ("stride_b", 40))}, **kw})
    assert nat.load().osm_gated_ema_step(ctypes.byref(a), None) == code


def block(**kw):
    fields = dict(rows=100, D=64, eps=1e-5, flags=nat.RESNORM_NORM_Y, stats=P)
    for n in ("x", "y", "gate", "r", "n"):
        fields[n], fields[n + "_stride"] = P, 64
    return made(nat.ResnormArgs, **{**fields, **kw})


BLOCK_ERRORS = [(dict(abi_version=1), -1), (dict(flags=4), -1), (dict(stream_dtype=2), -3), (dict(stream_dtype=1), -3), (dict(block_dtype=3), -3),
                (dict(rows=-1), -2), (dict(D=0), -2), (dict(D=1 << 31), -2), (dict(eps=-1.0), -1), (dict(eps=float("nan")), -1),
                (dict(x=None), -1), (dict(y=P + 2), -4), (dict(gate_stride=-64), -4), (dict(scale=P + 1), -4), (dict(weight=P + 2), -4),
                (dict(bias=P + 2), -4), (dict(stats=P + 2), -4)]


@pytest.mark.parametrize("kw,code", BLOCK_ERRORS + [(dict(r=None), -1), (dict(n_stride=63), -4)])
def test_block_errors(kw, code):
    assert nat.load().osm_residual_norm_fwd(ctypes.byref(block(**kw)), None) == code


@pytest.mark.parametrize("kw,bwd,code", [(kw, {}, code) for kw, code in BLOCK_ERRORS] + [
    (dict(stats=None), {}, -1), (dict(gate=None), {}, -1), ({}, dict(grad_r=P + 2), -4), ({}, dict(grad_n=P + 2), -4),
    ({}, dict(grad_x_stride=63), -4), ({}, dict(grad_y_stride=0), -4), ({}, dict(grad_gate=P + 2), -4), ({}, dict(grad_scale=P + 2), -4)])
def test_block_backward_errors(kw, bwd, code):
    fields = {}
    for n in ("grad_r", "grad_n", "grad_x", "grad_y", "grad_gate"):
        fields[n], fields[n + "_stride"] = P, 64
    b = made(nat.ResnormBwdArgs, **{**fields, **bwd})
    assert nat.load().osm_residual_norm_bwd(ctypes.byref(block(**kw)), ctypes.byref(b), ctypes.c_void_p(P), 1 << 40, None) == code


def test_block_workspace():
    lib = nat.load()
    need = lib.osm_residual_norm_bwd_workspace_bytes(ctypes.byref(block()))
    assert need == 25 * 3 * 64 * 4               # a line of sums for four rows
    assert lib.osm_residual_norm_bwd_workspace_bytes(ctypes.byref(block(rows=0))) == 0
    assert lib.osm_residual_norm_bwd_workspace_bytes(ctypes.byref(block(D=8193))) == (25 * 3 * 8193 + 200) * 4
    b = made(nat.ResnormBwdArgs)
    for ws, n in ((None, need), (P + 16, need), (P, need - 1)):
        assert lib.osm_residual_norm_bwd(ctypes.byref(block()), ctypes.byref(b), ctypes.c_void_p(ws), n, None) == -5
    assert lib.osm_residual_norm_bwd(ctypes.byref(block()), None, None, 0, None) == -1


def loss(**kw):
    return made(nat.LossArgs, **{**dict(N=100, D=64, V=500, hidden=P, hidden_stride=64, weight=P, weight_stride=64, targets=P, losses=P,
                                        lse=P), **kw})


LOSS_ERRORS = COMMON + [(dict(N=-1), -2), (dict(N=1 << 21), -2), (dict(D=0), -2), (dict(D=1 << 18), -2), (dict(V=0), -2), (dict(V=1 << 29), -2),
                        (dict(hidden=None), -1), (dict(weight=P + 2), -4), (dict(weight_stride=-1), -4), (dict(hidden_stride=-64), -4),
                        (dict(targets=None), -1), (dict(targets=P + 4), -1), (dict(lse=None), -1), (dict(lse=P + 2), -1)]


@pytest.mark.parametrize("kw,code", LOSS_ERRORS + [(dict(losses=P + 2), -4), (dict(loss=P + 2), -4), (dict(count=P + 1), -4), (dict(losses=None, loss=P), -1),
                                                   (dict(count=P), -1), (dict(flags=2), -1)])
def test_loss_errors(kw, code):
    assert nat.load().osm_linear_ce_fwd(ctypes.byref(loss(**kw)), ctypes.c_void_p(P), 1 << 40, None) == code


@pytest.mark.parametrize("kw,bwd,code", [(kw, {}, code) for kw, code in LOSS_ERRORS] + [
    ({}, dict(grad=P + 2), -4), ({}, dict(grad_losses=P + 2), -4), ({}, dict(count=P + 1), -4), ({}, dict(grad_hidden=P + 4), -4),
    ({}, dict(grad_weight=P + 8), -4), (dict(D=63), dict(grad_weight=P + 2), -4)])
def test_loss_backward_errors(kw, bwd, code):
    b = nat.LossBwdArgs()
    for k, v in {**dict(grad_hidden=P, grad_weight=P), **bwd}.items():
        setattr(b, k, v)
    assert nat.load().osm_linear_ce_bwd(ctypes.byref(loss(**kw)), ctypes.byref(b), ctypes.c_void_p(P), 1 << 40, None) == code


def test_loss_workspace():
    lib = nat.load()
    b = nat.LossBwdArgs()
    for size, call in ((lib.osm_linear_ce_workspace_bytes, lambda w, n: lib.osm_linear_ce_fwd(ctypes.byref(loss()), w, n, None)),
                       (lib.osm_linear_ce_bwd_workspace_bytes,
                        lambda w, n: lib.osm_linear_ce_bwd(ctypes.byref(loss()), ctypes.byref(b), w, n, None))):
        need = size(ctypes.byref(loss()))
        assert need > 0 and size(ctypes.byref(loss(N=0))) == 0 and size(ctypes.byref(loss(V=0))) == 0
        for ws, n in ((None, need), (P + 16, need), (P, need - 1)):
            assert call(ctypes.c_void_p(ws), n) == -5
    assert lib.osm_linear_ce_bwd(ctypes.byref(loss()), None, None, 0, None) == -1
    # the backward's memory is bounded by a piece's, whatever the vocabulary (fp32: six times 2^27 elements of P's parts)
    at = [lib.osm_linear_ce_bwd_workspace_bytes(ctypes.byref(loss(N=1 << 15, V=v, dtype=1))) for v in (1 << 15, 1 << 25)]
    assert max(at) < 2 * (1 << 27) * 2 + (64 << 20)


def test_no_cpu_path():
    x = torch.zeros(2, 3, 4)
    for call in (lambda: gated_ema(x, x), lambda: gated_ema_step(x[0], x[0], x[0]), lambda: residual_norm(x, x),
                 lambda: linear_cross_entropy(x, x[0], torch.zeros(2, 3, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="ROCm GPU only"):
            call()


@pytest.mark.parametrize("cls,cname", [(nat.Seq, "osm_seq"), (nat.EmaArgs, "osm_ema_args"), (nat.EmaBwdArgs, "osm_ema_bwd_args"),
                                       (nat.EmaStepArgs, "osm_ema_step_args"), (nat.ResnormArgs, "osm_resnorm_args"),
                                       (nat.ResnormBwdArgs, "osm_resnorm_bwd_args"), (nat.LossArgs, "osm_loss_args"),
                                       (nat.LossBwdArgs, "osm_loss_bwd_args")])
def test_struct_layout_matches_ctypes(cls, cname):
    from test_abi import test_struct_layout_matches_ctypes as layout
    layout(cls, cname)
