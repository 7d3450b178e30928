"""CPU checks of the layer norm's and the clipping's C entry points: sizes and
refusals, which come back as status codes before any HIP call."""
import ctypes

import pytest
import torch

from orthossm_amd import _native as nat
from orthossm_amd import clip_grad_norm, layer_norm


@pytest.fixture(autouse=True)
def _no_message_left():
    """A call that succeeds clears the thread's message."""
    yield
    a = nat.NormArgs()
    a.abi_version, a.D = nat.ABI_VERSION, 1
    assert nat.load().osm_layer_norm_fwd(ctypes.byref(a), None) == 0


def _norm(**kw):
    a = nat.NormArgs()
    a.abi_version, a.rows, a.D, a.eps = nat.ABI_VERSION, 100, 64, 1e-5
    a.x = a.y = a.mean = a.rstd = 0x10000      # never dereferenced: every case is refused
    a.x_stride = a.y_stride = 64
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(abi_version=1), -1), (dict(dtype=3), -3), (dict(rows=-1), -2), (dict(D=0), -2), (dict(D=1 << 31), -2),
    (dict(eps=-1.0), -1), (dict(eps=float("nan")), -1), (dict(x=None), -1), (dict(x=0x10002), -4), (dict(x_stride=-64), -4),
    (dict(y=None), -1), (dict(y_stride=63), -4), (dict(weight=0x10001), -4), (dict(mean=None), -1),
])
def test_norm_errors(kw, code):
    lib = nat.load()
    assert lib.osm_layer_norm_fwd(ctypes.byref(_norm(**kw)), None) == code
    assert lib.osm_last_error() != b""


def test_norm_backward_errors():
    lib = nat.load()

    def bwd(a, ws=0x10000, nbytes=1 << 30, **kw):
        b = nat.NormBwdArgs()
        b.grad_y, b.grad_y_stride = 0x10000, 64
        for k, v in kw.items():
            setattr(b, k, v)
        return lib.osm_layer_norm_bwd(ctypes.byref(a), ctypes.byref(b), ctypes.c_void_p(ws), nbytes, None)

    need = lib.osm_layer_norm_bwd_workspace_bytes(ctypes.byref(_norm()))
    assert need == 25 * 2 * 64 * 4               # a line of sums for four rows
    assert lib.osm_layer_norm_bwd_workspace_bytes(ctypes.byref(_norm(rows=0))) == 0
    assert bwd(_norm(mean=None, rstd=None)) == -1
    assert bwd(_norm(), None) == -5 and bwd(_norm(), 0x10010) == -5 and bwd(_norm(), nbytes=need - 1) == -5
    assert bwd(_norm(), grad_y=None) == -1 and bwd(_norm(), grad_x=0x10000, grad_x_stride=60) == -4
    assert bwd(_norm(), grad_weight=0x10002) == -4


def _clip(sizes=(5, 70000), dtypes=(0, 1), pointers=(0x10000, 0x20000), **kw):
    n = len(sizes)
    a = nat.ClipArgs()
    a.abi_version, a.count, a.flags, a.max_norm, a.norm = nat.ABI_VERSION, n, nat.CLIP_SCALE, 1.0, 0x30000
    a.tensors = (ctypes.c_void_p * n)(*pointers)
    a.sizes = (ctypes.c_int64 * n)(*sizes)
    a.dtypes = (ctypes.c_int32 * n)(*dtypes)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_clip_sizes():
    lib = nat.load()
    assert lib.osm_clip_workspace_bytes(ctypes.byref(_clip())) == (1 + 9) * 8       # chunks of 8192 elements
    assert lib.osm_clip_workspace_bytes(ctypes.byref(_clip((0, 1 << 35)))) == 1024 * 8
    assert lib.osm_clip_workspace_bytes(ctypes.byref(_clip((), (), ()))) == 8
    many = _clip((1,) * 301, (0,) * 301, (0x10000,) * 301)                           # three launches
    assert lib.osm_clip_workspace_bytes(ctypes.byref(many)) == 301 * 8


@pytest.mark.parametrize("args,kw,code", [
    ({}, dict(abi_version=0), -1), ({}, dict(flags=2), -1), ({}, dict(count=-1), -2), ({}, dict(count=1 << 30), -2),
    ({}, dict(max_norm=-1.0), -1), ({}, dict(eps=float("nan")), -1), ({}, dict(norm=None), -1), ({}, dict(norm=0x30002), -1),
    (dict(dtypes=(0, 2)), {}, -3), (dict(sizes=(5, -1)), {}, -2), (dict(sizes=(1 << 41, 1)), {}, -2),
    (dict(pointers=(0x10000, None)), {}, -1), (dict(pointers=(0x10002, 0x20000)), {}, -4),
    (dict(pointers=(0x10000, 0x20001)), {}, -4),
])
def test_clip_errors(args, kw, code):
    lib = nat.load()
    assert lib.osm_clip_grad_norm(ctypes.byref(_clip(**args, **kw)), ctypes.c_void_p(0x40000), 1 << 20, None) == code


def test_clip_workspace_errors():
    lib = nat.load()
    for ws, n in ((None, 80), (0x40010, 80), (0x40000, 79)):
        assert lib.osm_clip_grad_norm(ctypes.byref(_clip()), ctypes.c_void_p(ws), n, None) == -5


def test_no_cpu_path():
    with pytest.raises(RuntimeError, match="ROCm GPU only"):
        layer_norm(torch.zeros(2, 4))
    with pytest.raises(RuntimeError, match="ROCm GPU only"):
        clip_grad_norm([torch.zeros(4)], 1.0)


@pytest.mark.parametrize("cls,cname", [(nat.NormArgs, "osm_norm_args"), (nat.NormBwdArgs, "osm_norm_bwd_args"),
                                      (nat.ClipArgs, "osm_clip_args")])
def test_struct_layout_matches_ctypes(cls, cname):
    from test_abi import test_struct_layout_matches_ctypes as layout
    layout(cls, cname)


def test_clip_refuses_tensors_that_share_memory():
    """(workspace errors, -5, come after; nothing is launched)"""
    lib = nat.load()

    def clip(sizes, dtypes, pointers, **kw):
        return lib.osm_clip_grad_norm(ctypes.byref(_clip(sizes, dtypes, pointers, **kw)), None, 0, None)

    for sizes, dtypes, pointers in (((5, 5), (0, 0), (0x10000, 0x10000)), ((5, 5), (0, 0), (0x10000, 0x10010)),
                                    ((5, 5), (0, 0), (0x10010, 0x10000)), ((9, 1), (1, 1), (0x10000, 0x10010)),
                                    ((100, 1, 1), (0, 1, 0), (0x10000, 0x10004, 0x20000))):
        assert clip(sizes, dtypes, pointers) == -4
        assert b"share memory" in lib.osm_last_error()
        assert clip(sizes, dtypes, pointers, flags=0) == -5          # the norm alone only reads
    for sizes, dtypes, pointers in (((5, 5), (0, 0), (0x10000, 0x10014)), ((8, 1), (1, 0), (0x10000, 0x10010)),
                                    ((5, 0, 0), (0, 0, 1), (0x10000, 0x10004, 0x10000))):
        assert clip(sizes, dtypes, pointers) == -5


def test_shared_memory_of_tensors():
    from orthossm_amd.grad_clip import _share_memory

    flat = torch.zeros(240)
    square = flat.view(4, 60)
    shared = ([flat, flat[1:]], [flat[5:9], flat[:6]], [flat, square.t()], [square[:, ::2], square[:, ::2]],
              [square[:, ::2], flat[:1]], [square[:, 1::2], flat[235:]], [flat[:3].expand(2, 3)], [flat[:1].expand(5)])
    apart = ([flat[:5], flat[5:]], [square[:, ::2], square[:, 1::2]], [square[:, :5], square[:, 5:]],
             [flat[10:20], flat[30:40].view(2, 5).t(), flat[:10]], [flat[:1], flat[1:2]], [])
    for tensors in shared:
        assert _share_memory(tensors) and _share_memory(tensors[::-1])
    for tensors in apart:
        assert not _share_memory(tensors) and not _share_memory(tensors[::-1])
