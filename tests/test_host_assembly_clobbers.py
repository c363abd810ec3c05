"""Assembly in the kernels names the special registers that it writes: the compiler would keep numbers of its own there otherwise."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dihydrogen_amd", "csrc")


STRING = re.compile(r'"((?:[^"\\]|\\.)*)"')


def _statements(text):
    """Of each asm statement the template, and the clobbers, which are its fourth part."""
    for m in re.finditer(r"\basm\b\s*(?:volatile\s*)?\(", text):
        depth, end = 1, m.end()
        while depth:
            depth += {"(": 1, ")": -1}.get(text[end], 0)
            end += 1
        body = text[m.end():end - 1]
        strings = iter(STRING.findall(body))
        parts = [[next(strings) for _ in re.findall('""', part)] for part in STRING.sub('""', body).split(":")]
        yield "".join(parts[0]), set(parts[3]) if len(parts) > 3 else set()


def _written(template):
    """Special registers that stand as an instruction's first operand."""
    return set(re.findall(r"\bs_\w+\s+(m0|vcc|exec|scc)\b", template.replace("\\n", "\n").replace("\\t", "\t")))


@pytest.mark.parametrize("path", sorted(glob.glob(os.path.join(CSRC, "*.h*"))), ids=os.path.basename)
def test_special_registers_are_named(path):
    for template, clobbers in _statements(open(path).read()):
        assert _written(template) <= clobbers, template


def test_statements_are_found():
    text = 'asm volatile("s_mov_b32 m0, %0\\n\\ts_nop 4" ::"s"(f(x)) : "memory", "m0"); asm("s_mov_b64 vcc, 0"); asm volatile("" : "+a"(v));'
    found = list(_statements(text))
    assert [(_written(t), c) for t, c in found] == [({"m0"}, {"memory", "m0"}), ({"vcc"}, set()), (set(), set())]
