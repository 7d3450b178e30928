"""CPU checks of the gated delta rule: the oracle's gradients against central
differences, and the C entry points' refusals (status codes before any HIP
call)."""
import ctypes

import pytest
import torch

from oracle import delta as O
from orthossm_amd import _native as nat
from orthossm_amd import gated_delta_forward


@pytest.fixture(autouse=True)
def _no_message_left():
    """A call that succeeds clears the thread's message."""
    yield
    a = nat.DeltaStepArgs()
    a.abi_version, a.H, a.Hk, a.dk, a.dv = nat.ABI_VERSION, 1, 1, 1, 1
    assert nat.load().osm_delta_step(ctypes.byref(a), None) == 0


def test_oracle_gradients_against_differences():
    gen = torch.Generator().manual_seed(0)
    B, S, H, Hk, dk, dv = 2, 6, 4, 2, 3, 5

    def rand(*shape):
        return torch.randn(*shape, generator=gen, dtype=torch.float64)

    t = [rand(B, S, Hk, dk), rand(B, S, Hk, dk), rand(B, S, H, dv), -rand(B, S, H).abs(), rand(B, S, H), rand(B, H, dk, dv)]
    go, gs, lengths = rand(B, S, H, dv), rand(B, H, dk, dv), torch.tensor([6, 4])
    grads = O.gated_delta_grads(*t[:5], go, gs, state_init=t[5], lengths=lengths)[2:]

    def loss(u):
        out, fin = O.gated_delta(*u[:5], state_init=u[5], lengths=lengths)
        return ((out * go).sum() + (fin * gs).sum()).item()

    h = 1e-5
    for i, grad in enumerate(grads):
        way = rand(*t[i].shape)
        up, down = (loss([x + s * h * way if j == i else x for j, x in enumerate(t)]) for s in (1, -1))
        assert abs((up - down) / (2 * h) - (grad * way).sum().item()) <= 1e-6 * (1 + grad.norm().item())


def test_no_cpu_path():
    x = torch.zeros(1, 4, 1, 8)
    with pytest.raises(RuntimeError, match="ROCm GPU only"):
        gated_delta_forward(x, x, x, x[..., 0], x[..., 0])


def _args(**kw):
    a = nat.DeltaArgs()
    a.abi_version = nat.ABI_VERSION
    a.B, a.S, a.H, a.Hk, a.dk, a.dv = 2, 200, 4, 2, 48, 80
    for r, (s, h) in ((a.q, (96, 48)), (a.k, (96, 48)), (a.v, (320, 80)), (a.out, (320, 80)), (a.g, (4, 1)),
                      (a.beta, (4, 1))):
        r.p, r.stride_b, r.stride_s, r.stride_h = 0x10000, 200 * s, s, h   # never dereferenced here
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _fwd(a, ws=None, nbytes=0):
    return nat.load().osm_delta_fwd(ctypes.byref(a), ctypes.c_void_p(ws), nbytes, None)


def test_sizes():
    lib = nat.load()
    chunks = 2 * 4 * 4                      # rows, heads, chunks of 64 tokens
    solved, states = (chunks * n * 4 for n in (48 * 64 + 320, 64 * 80))                 # 48 rows of a state held as 64
    segments = 2 * 4 * 4 * (64 * 64 + 64 * 80) * 4                                      # four of one chunk a row
    assert lib.osm_delta_saved_bytes(ctypes.byref(_args())) == solved + states
    assert lib.osm_delta_workspace_bytes(ctypes.byref(_args())) == solved + segments
    assert lib.osm_delta_workspace_bytes(ctypes.byref(_args(saved=0x10000))) == segments
    assert lib.osm_delta_workspace_bytes(ctypes.byref(_args(S=8))) == 0       # token by token
    assert lib.osm_delta_workspace_bytes(ctypes.byref(_args(S=9))) > 0
    assert lib.osm_delta_workspace_bytes(ctypes.byref(_args(S=0))) == 0
    # the backward: maps of the segments, the chunks' gradients, and a gradient of q and k for each of v's heads
    assert lib.osm_delta_bwd_workspace_bytes(ctypes.byref(_args())) == segments + states + 2 * 2 * 200 * 4 * 48 * 4
    assert lib.osm_delta_bwd_workspace_bytes(ctypes.byref(_args(Hk=4))) == segments + states


@pytest.mark.parametrize("kw,code", [
    (dict(abi_version=1), -1), (dict(dtype=2), -3), (dict(B=-1), -2), (dict(S=-1), -2), (dict(S=(1 << 31) - 64), -2),
    (dict(H=3), -2), (dict(Hk=0), -2), (dict(dk=0), -2), (dict(dk=129), -2), (dict(dv=0), -2), (dict(dv=1 << 20), -2),
    (dict(B=1 << 20, S=1 << 20), -2), (dict(H=1 << 20, Hk=1 << 20), -2), (dict(lengths=0x10002), -4),
    (dict(state_init=0x10001), -4), (dict(state_out=0x10002), -4), (dict(saved=0x10010), -5),
])
def test_argument_errors(kw, code):
    assert _fwd(_args(**kw)) == code
    assert nat.load().osm_last_error() != b""


@pytest.mark.parametrize("name", ["q", "k", "v", "out", "g", "beta"])
def test_row_errors(name):
    for field, value, code in (("p", None, -1), ("p", 0x10001, -4), ("stride_b", -1, -4), ("stride_s", -4, -4),
                               ("stride_h", -8, -4)):
        a = _args()
        setattr(getattr(a, name), field, value)
        assert _fwd(a) == code, (field, value)


def test_workspace_errors():
    need = nat.load().osm_delta_workspace_bytes(ctypes.byref(_args()))
    assert _fwd(_args()) == -5
    assert _fwd(_args(), 0x10000, need - 1) == -5
    assert _fwd(_args(), 0x10010, need) == -5


def test_backward_errors():
    lib = nat.load()
    b = nat.DeltaBwdArgs()

    def bwd(a, b, ws=None, nbytes=0):
        return lib.osm_delta_bwd(ctypes.byref(a), ctypes.byref(b) if b is not None else None, ctypes.c_void_p(ws), nbytes,
                                 None)

    assert bwd(_args(), None) == -1
    assert bwd(_args(), b) == -1                            # nothing saved
    assert bwd(_args(saved=0x10000), b) == -1               # no grad_out
    for name in ("grad_out", "grad_q", "grad_k", "grad_v", "grad_g", "grad_beta"):
        getattr(b, name).p, getattr(b, name).stride_s = 0x10000, 320
    assert bwd(_args(saved=0x10000), b) == -5
    b.grad_init = 0x10002
    assert bwd(_args(saved=0x10000), b) == -4
    b.grad_init, b.grad_q.stride_s = None, 47               # rows of 48 overlap
    assert bwd(_args(saved=0x10000), b) == -4
    assert _fwd(_args(v=nat.Rows(0x10000, 200 * 320, 79, 80))) == -4


def test_step_errors():
    lib = nat.load()

    def step(**kw):
        a = nat.DeltaStepArgs()
        a.abi_version = nat.ABI_VERSION
        a.B, a.H, a.Hk, a.dk, a.dv, a.n_slots = 2, 4, 2, 48, 80, 3
        a.state, a.state_stride = 0x10000, 4 * 48 * 80
        for r in (a.q, a.k, a.v, a.out, a.g, a.beta):
            r.p = 0x10000
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.osm_delta_step(ctypes.byref(a), None)

    for kw, code in ((dict(abi_version=0), -1), (dict(dtype=9), -3), (dict(H=5), -2), (dict(dk=200), -2),
                     (dict(n_slots=1), -2), (dict(n_slots=-1), -2), (dict(state=None), -1), (dict(state=0x10002), -4),
                     (dict(slots=0x10004), -4), (dict(state_stride=100), -4), (dict(q=nat.Rows()), -1),
                     (dict(beta=nat.Rows(0x10002, 0, 0, 0)), -4)):
        assert step(**kw) == code, kw


@pytest.mark.parametrize("cls,cname", [(nat.Rows, "osm_rows"), (nat.DeltaArgs, "osm_delta_args"),
                                      (nat.DeltaBwdArgs, "osm_delta_bwd_args"), (nat.DeltaStepArgs, "osm_delta_step_args")])
def test_struct_layout_matches_ctypes(cls, cname):
    from test_abi import test_struct_layout_matches_ctypes as layout
    layout(cls, cname)


def test_a_single_tokens_stride_is_not_checked():
    """The errors are those of a later argument, not of the strides."""
    lib = nat.load()
    for stride in (1 << 40, 0, -4):
        a = _args(S=1, saved=0x10010)
        for name in ("q", "k", "v", "g", "beta"):
            getattr(a, name).stride_s = stride
        assert _fwd(a) == -5
        s = nat.DeltaStepArgs()
        s.abi_version = nat.ABI_VERSION
        s.B, s.H, s.Hk, s.dk, s.dv, s.n_slots = 2, 4, 2, 48, 80, 3
        for r in (s.q, s.k, s.v, s.out, s.g, s.beta):
            r.p, r.stride_s = 0x10000, stride
        assert lib.osm_delta_step(ctypes.byref(s), None) == -1
        assert lib.osm_last_error() == b"state is NULL"


@pytest.mark.parametrize("dtype,S", [(torch.int8, 200), (torch.uint8, 5001), (torch.int16, 40000), (torch.int64, 1 << 30),
                                     (torch.uint16, 70000), (torch.int32, 100)])
def test_lengths_of_a_type_that_does_not_hold_the_sequence(dtype, S):
    from orthossm_amd.delta import _lengths

    got = _lengths(torch.tensor([3, 0, 100], dtype=dtype), 3, S, torch.device("cpu"))
    assert got.dtype == torch.int32 and got.tolist() == [3, 0, 100]


def test_lengths_past_32_bits():
    from orthossm_amd.delta import _lengths

    assert _lengths(torch.tensor([1 << 40, -1 << 40, 7]), 3, 50, torch.device("cpu")).tolist() == [50, 0, 7]


def test_outputs_lie_in_no_arguments_memory():
    from orthossm_amd.delta import apart

    flat = torch.zeros(240)
    x, out = flat[:120].view(10, 12), flat[120:].view(10, 12)
    apart("out", out, dict(x=x, w=None, none=flat[:0]), "x")
    apart("out", x, dict(x=x, y=out), "x")
    apart("out", x, dict(x=flat[:120].view(10, 12)), "x")
    for others in (dict(y=x), dict(x=flat[1:121].view(10, 12)), dict(x=flat[:100].view(10, 10)), dict(y=out, z=flat[119:130]),
                   dict(x=flat[:144].view(12, 12)[:10, :].t()), dict(x=x.view(12, 10).t()), dict(y=flat[::3])):
        with pytest.raises(ValueError, match="out shares memory with"):
            apart("out", x, others, "x")
