"""Checks on the inline assembly of the kernels' sources (CPU only)."""
import os
import re

from orthossm_amd import build as B

ASM = re.compile(r"\basm\s+(?:volatile\s*)?\((.*?)\)\s*;", re.S)
WRITES_M0 = re.compile(r"\bs_\w+\s+m0\b")


def undeclared(source):
    """The asm statements that write M0 and do not say so among their clobbers."""
    found = []
    for m in ASM.finditer(source):
        code, _, rest = m.group(1).partition(":")
        if WRITES_M0.search(code) and '"m0"' not in rest:
            found.append(m.group(0))
    return found


def test_detector():
    text = 'asm volatile("s_mov_b32 m0, %1\\n\\tglobal_load_lds_dwordx4 %0, off" ::"v"(a), "s"(b) : "memory"{});'
    assert len(undeclared(text.format(""))) == 1 and undeclared(text.format(', "m0"')) == []
    assert undeclared('asm volatile("v_mov_b32 v0, m0" ::: "v0");') == []


def test_writes_to_m0_are_declared():
    """The compiler keeps values in M0 across statements that it takes to leave
    the register alone."""
    for name in sorted(os.listdir(B.CSRC)):
        with open(os.path.join(B.CSRC, name)) as f:
            assert undeclared(f.read()) == [], name
