"""Wait states in the kernels' inline assembly.  Inside one asm statement the
compiler inserts none, so a load to LDS that follows a scalar write of its
address register m0 needs its s_nop written out (the compiler puts one between
the two where it writes them itself)."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(__file__), "..", "nativebit_amd", "csrc")


def statements(text):
    """The instructions of every asm statement."""
    for m in re.finditer(r"\basm\s*(?:volatile)?\s*\(\s*((?:\"(?:[^\"\\]|\\.)*\"\s*)+)", text):
        code = "".join(re.findall(r"\"((?:[^\"\\]|\\.)*)\"", m.group(1)))
        yield [i.strip() for i in re.split(r"\\n|\\t|;", code) if i.strip()]


def early(code):
    """Loads to LDS with no wait state after a write of m0 in the same statement."""
    return [b for a, b in zip(code, code[1:])
            if re.match(r"s_\w+ m0\b", a) and re.search(r"load_lds|\blds\b", b)]


def test_the_rule_finds_the_pair():
    bad = 'asm volatile("s_mov_b32 m0, %0\\n\\tglobal_load_lds_dwordx4 %1, off" : : "s"(a));'
    good = 'asm volatile("s_mov_b32 m0, %0\\n\\t"\n"s_nop 0\\n\\tglobal_load_lds_dwordx4 %1, off" : : "s"(a));'
    assert [early(c) for c in statements(bad)] == [["global_load_lds_dwordx4 %1, off"]]
    assert [early(c) for c in statements(good)] == [[]]


@pytest.mark.parametrize("name", sorted(f for f in os.listdir(CSRC) if f.endswith((".h", ".hip"))))
def test_loads_to_lds_wait_for_m0(name):
    with open(os.path.join(CSRC, name)) as f:
        found = list(statements(f.read()))
    assert not [b for code in found for b in early(code)]


def test_the_loads_are_seen():
    """The statements that the rule is for are found in the sources."""
    seen = 0
    for name in os.listdir(CSRC):
        if name.endswith((".h", ".hip")):
            with open(os.path.join(CSRC, name)) as f:
                seen += sum("load_lds" in i for code in statements(f.read()) for i in code)
    assert seen >= 5
