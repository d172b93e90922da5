"""Inline assembly of the kernels lists the registers that it writes by name as clobbers: the
compiler takes any other to keep its value."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "pagoda_amd" / "csrc"
SOURCES = sorted(p.name for p in CSRC.iterdir() if "asm volatile" in p.read_text())


def statements(text):
    """(template, clobbers) of every asm statement."""
    for m in re.finditer(r'asm volatile\(((?:"(?:[^"\\]|\\.)*"|[^";])*)\);', text):
        part, parts = 0, ["", "", "", ""]
        for token in re.findall(r'"(?:[^"\\]|\\.)*"|:|[^":]+', m.group(1)):
            if token == ":":
                part += 1
            elif token[0] == '"':
                parts[part] += token + " "
        yield parts[0], parts[3]


def test_statements_are_found():
    got = list(statements('asm volatile("s_mov_b32 m0, %0" ::"s"(x(1)) : "memory", "m0");\n  asm volatile("" ::: "memory");'))
    assert got == [('"s_mov_b32 m0, %0" ', '"memory" "m0" '), ('"" ', '"memory" ')]


@pytest.mark.parametrize("name", SOURCES)
def test_named_registers_are_clobbers(name):
    text = (CSRC / name).read_text()
    found = list(statements(text))
    assert len(found) == text.count("asm volatile")
    for template, clobbers in found:
        for reg in re.findall(r"\b[sv]_\w+ (m0|vcc|exec|[sv]\d+),", template):
            assert f'"{reg}"' in clobbers, template
