"""The workspaces of the vocabulary's cross entropy (CPU only): bounded by the
pieces that the vocabulary is taken in, whichever operand a piece's copy is of."""
import ctypes

import pytest

from orthossm_amd import _native as nat

P = 0x10000      # never dereferenced
PIECE = 9 * (1 << 24) * 2      # bytes of a piece's parts of P, or of its copied weights


def args(N, D, V, dtype, shift=0, gap=0):
    """shift: bytes of the weights' address past 16; gap: elements between their rows."""
    a = nat.LossArgs()
    for k, v in dict(abi_version=nat.ABI_VERSION, dtype=dtype, N=N, D=D, V=V, hidden=P, hidden_stride=D, weight=P + shift,
                     weight_stride=D + gap, targets=P, losses=P, lse=P).items():
        setattr(a, k, v)
    return ctypes.byref(a)


def up(n, to):
    return (n + to - 1) // to * to


# dtype, shift, gap, columns less than a multiple of 64: weights that are copied (fp32, or rows that are
# no whole units, or not aligned), and not
COPIED = [(0, 0, 0, 0), (1, 0, 0, 1), (1, 2, 0, 0), (1, 0, 4, 0)]
FORMS = [(form, True) for form in COPIED] + [((1, 0, 0, 0), False)]


@pytest.mark.parametrize("N", [1, 64, 256, 3000, 1 << 15])
@pytest.mark.parametrize("form,copied", FORMS)
def test_backward_is_bounded_by_its_pieces(form, copied, N):
    """Beside the hidden rows' copy and their sums: P and the copied weights of a piece."""
    dtype, shift, gap, less = form
    parts = 1 if dtype else 3
    for width in (64, 1024, 4096, 1 << 14):
        n, d = up(N, 256), width
        sums = 4 * n * d * max(1, min(8, 256 // (up(d, 256) // 256 * (n // 256))))
        most = 2 * parts * n * d + sums + max(PIECE, 2 * n * 256 * max(parts, 2)) + (1 << 20)
        if copied:
            most += max(PIECE, 2 * 256 * d * parts)
        for V in (30000, 128256, 1 << 18, 1 << 25):
            need = nat.load().osm_linear_ce_bwd_workspace_bytes(args(N, width - less, V, dtype, shift, gap))
            assert 0 < need <= most, (N, width, V)


@pytest.mark.parametrize("N", [1, 64, 65, 5000])
@pytest.mark.parametrize("form", COPIED)
def test_copies_are_of_fewer_threads_than_a_launch_may_have(form, N):
    """A thread copies 8 columns of a class, 16 bytes a part."""
    dtype, shift, gap, less = form
    for width in (1 << 14, 1 << 17):
        need = nat.load().osm_linear_ce_bwd_workspace_bytes(args(N, width - less, 1 << 28, dtype, shift, gap))
        assert 0 < need / (16 * (1 if dtype else 3)) < 1 << 32


@pytest.mark.parametrize("dtype", [0, 1])
def test_statistics_are_of_the_tiles_that_there_are(dtype):
    """8 bytes a token and tile: of 256 classes in bf16 and 128 in fp32 where there are many."""
    N, D, V = 1 << 16, 64, 128000
    n, parts, rows = N, 1 if dtype else 3, 256 if dtype else 128
    copies = 2 * parts * n * D + (0 if dtype else 2 * parts * up(V, 256) * D)
    need = nat.load().osm_linear_ce_workspace_bytes(args(N, D, V, dtype))
    assert need <= 8 * n * (up(V, rows) // rows) + copies + 16 * n + (1 << 16)
