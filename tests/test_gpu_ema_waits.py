"""The waits of the gated EMA's tiles for those ahead of them: past one group of
tiles where tiles go by index (lane-blocks a multiple of 8) and where they are
drawn, and states and their gradients in place."""
import ctypes

import pytest
import torch
from test_gpu_gated_ema import check, make

from orthossm_amd import _native as nat
from orthossm_amd import ema, gated_ema_backward, gated_ema_forward

pytestmark = pytest.mark.gpu

# By index: 8, 8 and 16 lane-blocks; drawn: 6 and 9.  3000 tokens are 24 tiles, 3 groups forward, and 47, 6, backward.
INDEXED = [(8, 128), (4, 256), (8, 200)]
DRAWN = [(3, 256), (9, 100)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,D", INDEXED + DRAWN)
def test_groups_of_tiles(dev, B, D, dtype):
    check(dev, *make(B, 3000, D, dtype, seed=B + D))


@pytest.mark.parametrize("B,D", INDEXED + DRAWN)
def test_rows_of_different_lengths(dev, B, D):
    lengths = [3000, 0, 1025, 1024, 2047, 1, 129, 2999, 513][:B]
    check(dev, *make(B, 3000, D, seed=D), lengths=lengths)


def backward_in_place(x, gate, go, init, gs, lens=None):
    """dx, dgate, and dinit where dL/d state was, through the C entry point."""
    lib = nat.load()
    a, keep = ema._prepare(x, gate, init, lens)
    _, _, saved, _ = ema._forward(x, gate, init, lens, None, False, None, True)
    a.saved = saved.data_ptr()
    b = nat.EmaBwdArgs()
    grads = [torch.empty_like(x), torch.empty_like(x)]
    for name, t in zip(("grad_out", "grad_x", "grad_gate"), (go, *grads)):
        ema._set_seq(getattr(b, name), t)
    state = gs.clone()
    b.grad_state = b.grad_init = state.data_ptr()
    ws = torch.empty(lib.osm_gated_ema_bwd_workspace_bytes(ctypes.byref(a)), dtype=torch.uint8, device=x.device)
    nat.check(lib.osm_gated_ema_bwd(ctypes.byref(a), ctypes.byref(b), ctypes.c_void_p(ws.data_ptr()), ws.numel(),
                                    ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
    del keep
    return *grads, state


@pytest.mark.parametrize("B,D", INDEXED + DRAWN)
@pytest.mark.parametrize("S", [60, 400, 3000])
def test_states_and_their_gradients_in_place(dev, S, B, D):
    x, gate, init, go, gs = (t.to(dev) for t in make(B, S, D, seed=S))
    for lens in (None, torch.tensor([S, 0, S // 2, 1, S, 65, S, S, 7][:B], dtype=torch.int32, device=dev)):
        want, last = gated_ema_forward(x, gate, state_init=init, lengths=lens, return_state=True)
        grads = gated_ema_backward(x, gate, go, state_init=init, lengths=lens, grad_state=gs, need_init=True)
        for _ in range(5):
            state = init.clone()
            got = gated_ema_forward(x, gate, state_init=state, lengths=lens, state_out=state)
            assert torch.equal(got, want) and torch.equal(state, last)
            assert all(torch.equal(p, q) for p, q in zip(grads, backward_in_place(x, gate, go, init, gs, lens)))


@pytest.mark.parametrize("B,D", INDEXED[:2])
def test_two_streams_at_once(dev, B, D):
    ins = [[t.to(dev) for t in make(B, 9000, D, seed=s)] for s in (13, 14)]

    def run(i):
        return (*gated_ema_forward(*i[:2], state_init=i[2], return_state=True),
                *gated_ema_backward(*i[:2], i[3], state_init=i[2], grad_state=i[4], need_init=True))

    want = [run(i) for i in ins]
    streams = [torch.cuda.Stream(dev) for _ in ins]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for i, s in zip(ins, streams):
            with torch.cuda.stream(s):
                got.append(run(i))
    torch.cuda.synchronize()
    for k, g in enumerate(got):
        assert all(torch.equal(p, q) for p, q in zip(g, want[k % 2]))
