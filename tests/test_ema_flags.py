"""CPU checks of the test aid that the gated EMA's entry points take beside the
type, and of where it does not belong."""
import ctypes

import pytest
from test_ema_block_loss import P, ema, made, seqs

from orthossm_amd import _native as nat

AID = nat.FLAG_POLL_LIMIT_ZERO


@pytest.mark.parametrize("dtype", [0, 1])
def test_poll_limit_beside_the_type(dtype):
    lib, b = nat.load(), made(nat.EmaBwdArgs, **seqs("grad_out", "grad_x", "grad_gate"))
    for size in (lib.osm_gated_ema_saved_bytes, lib.osm_gated_ema_workspace_bytes, lib.osm_gated_ema_bwd_workspace_bytes):
        assert size(ctypes.byref(ema(dtype=dtype | AID))) == size(ctypes.byref(ema(dtype=dtype))) > 0
    # refused for what comes after the type
    for kw, code in (({"x.p": P + 1}, -4), ({"x.p": None}, -1), (dict(saved=P + 2), -4)):
        a = ema(dtype=dtype | AID, **kw)
        assert lib.osm_gated_ema_fwd(ctypes.byref(a), ctypes.c_void_p(P), 1 << 40, None) == code
        assert lib.osm_gated_ema_bwd(ctypes.byref(a), ctypes.byref(b), ctypes.c_void_p(P), 1 << 40, None) == code


@pytest.mark.parametrize("dtype", [2 | AID, AID << 1, nat.FLAG_TIMING_JITTER, -1])
def test_other_types_are_refused(dtype):
    lib, b = nat.load(), made(nat.EmaBwdArgs, **seqs("grad_out", "grad_x", "grad_gate"))
    a = ema(dtype=dtype)
    assert lib.osm_gated_ema_fwd(ctypes.byref(a), ctypes.c_void_p(P), 1 << 40, None) == -3
    assert lib.osm_gated_ema_bwd(ctypes.byref(a), ctypes.byref(b), ctypes.c_void_p(P), 1 << 40, None) == -3
    step = made(nat.EmaStepArgs, B=4, D=40, state=P, state_stride=40, n_slots=4, dtype=AID)
    assert lib.osm_gated_ema_step(ctypes.byref(step), None) == -3
