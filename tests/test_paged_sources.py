"""What the sources and the built kernels of the batched-cache operators must not hold; no GPU needed."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fastvideo_amd", "csrc")
FILES = ("attn_ragged.h", "attn_ragged.hip", "attn_rows.hip", "paged.hip")


def asm_statements(text):
    """The argument text of every asm statement."""
    for m in re.finditer(r"\basm\s+volatile\s*\(", text):
        depth, at = 1, m.end()
        while depth:
            depth += {"(": 1, ")": -1}.get(text[at], 0)
            at += 1
        yield text[m.end():at - 1]


def loads_into_registers(statement):
    """An asm load that returns its register before the data is there: a load that is neither LDS-DMA nor waited for in the same statement."""
    code = " ".join(re.findall(r'"((?:[^"\\]|\\.)*)"', statement.split("\n:")[0].split(" : ")[0]))
    load = re.search(r"\b(global|buffer|flat|scratch|s)_load_|\bds_read", code)
    return bool(load) and not re.search(r"\blds\b", code) and "s_waitcnt" not in code


@pytest.mark.parametrize("name", FILES)
def test_no_load_in_assembly_leaves_its_register_behind(name):
    text = open(os.path.join(CSRC, name)).read()
    assert not [s for s in asm_statements(text) if loads_into_registers(s)]


def test_the_rule_knows_such_a_load():
    assert loads_into_registers('"global_load_dwordx4 %0, %1, off" : "=a"(x) : "v"(p) : "memory"')
    assert not loads_into_registers('"global_load_dwordx4 %0, %1, off\\n\\ts_waitcnt vmcnt(0)" : "=a"(x) : "v"(p) : "memory"')
    assert not loads_into_registers('"buffer_load_dwordx4 %4, s[96:99], 0 offen lds" : : "v"(at) : "memory"')
    assert not loads_into_registers('"s_waitcnt vmcnt(0)" ::: "memory"')
