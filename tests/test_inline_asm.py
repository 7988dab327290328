"""Every register that a piece of inline asm writes by name is among its clobbers: hipcc keeps values of its own in m0, vcc, exec and scc."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "quickvideo_amd", "csrc")


def statements(text):
    for m in re.finditer(r"\basm\s+(?:volatile\s*)?\(|\basm\(", text):
        depth, end = 1, m.end()
        for t in re.finditer(r'"(?:[^"\\]|\\.)*"|[()]', text[m.end():]):
            depth += {"(": 1, ")": -1}.get(t.group(), 0)
            if depth == 0:
                end += t.start()
                break
        yield text[m.end():end]


def undeclared(stmt):
    strings = re.findall(r'"((?:[^"\\]|\\.)*)"', stmt)
    written = set(re.findall(r"(?:^|\\n\\t|\\n|;)\s*[sv]_\w+\s+(m0|vcc(?:_lo|_hi)?|exec(?:_lo|_hi)?)\b", strings[0])) if strings else set()
    clobbers = set(strings[1:])
    return sorted(r for r in written if not {r, r.split("_")[0]} & clobbers)


def test_the_check_sees_a_missing_clobber():
    assert undeclared(r'"s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" : : "s"(a), "v"(b), "s"(c) : "memory"') == ["m0"]
    assert undeclared(r'"s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" : : "s"(a), "v"(b), "s"(c) : "memory", "m0"') == []
    assert undeclared(r'"s_nop 1" ::') == [] and undeclared(r'"" : "+v"(x)') == []
    assert list(statements('x; asm volatile("a (%0) \\"" : "=v"(f(x)) : : "memory"); y(); asm("b" ::);')) == ['"a (%0) \\"" : "=v"(f(x)) : : "memory"', '"b" ::']


@pytest.mark.parametrize("path", sorted(glob.glob(os.path.join(CSRC, "*.hip")) + glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.inc"))),
                         ids=os.path.basename)
def test_named_registers_are_declared(path):
    with open(path) as f:
        bad = [(s.strip()[:80], undeclared(s)) for s in statements(f.read()) if undeclared(s)]
    assert not bad
