"""The gfx950 assembly of the gated EMA's, the residual norm's and the cross
entropy's kernels (CPU only): nothing stands between a store wider than 64 bits
and its wait states, those that the compiler made of narrower ones among them."""
import os
import re
import subprocess

import pytest
from test_isa import WIDE_STORE, instructions

from orthossm_amd import build as B


@pytest.mark.parametrize("name", ["osm_ema", "osm_resnorm", "osm_loss"])
def test_wide_stores_are_followed_by_their_wait(name, tmp_path):
    out = str(tmp_path / "kernels.s")
    subprocess.run(B.device_asm_command(os.path.join(B.CSRC, name + ".hip"), out), check=True, capture_output=True)
    with open(out) as f:
        ins = list(instructions(f.read()))
    assert any(WIDE_STORE.match(t) for t in ins)
    bad = [pair for pair in zip(ins, ins[1:]) if WIDE_STORE.match(pair[0]) and not re.match(r"s_nop [1-9]", pair[1])]
    assert bad == [], (len(bad), bad[:3])
