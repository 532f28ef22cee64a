"""Inline assembly of the device code names the registers that it writes (CPU only): what the compiler keeps in one
that is not named would be lost."""
from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "stagehand_amd" / "csrc"
ASM = re.compile(r"\basm\b(?:\s+volatile)?\s*\((.*?)\)\s*;", re.S)
# an instruction's first operand, where that is a register by name
WRITTEN = re.compile(r"(?:^|\\n\\t|\\n|;)\s*[sv]_(?!waitcnt|nop|barrier)\w+\s+(m0|vcc|exec|scc|[sv]\d+|[sv]\[\d+:\d+\])\b")


def statements():
    """(file, instructions, what stands behind them: outputs, inputs, clobbers)"""
    for path in sorted(CSRC.glob("*.hip")):
        for m in ASM.finditer(path.read_text()):
            text = re.match(r'\s*((?:"(?:[^"\\]|\\.)*"\s*)+)', m.group(1))
            if text:
                yield path.name, "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', text.group(1))), m.group(1)[text.end():]


def test_registers_that_are_written_by_name_are_declared():
    for name, text, operands in statements():
        for register in WRITTEN.findall(text):
            assert f'"{register}"' in operands, f"{name}: {text!r} writes {register} and does not say so"


def test_loads_to_lds_take_m0_from_the_compiler():
    loads = [(name, text, operands) for name, text, operands in statements() if re.search(r"\blds\b", text)]
    assert loads
    for name, text, operands in loads:
        assert '"{m0}"' in operands, f"{name}: {text!r} reads M0, which is not among its inputs"


@pytest.mark.parametrize("line,writes", [("s_mov_b32 m0, %0\\n\\ts_nop 0", ["m0"]), ("s_waitcnt vmcnt(%0)", []),
                                         ("v_mov_b32 v3, 0", ["v3"]), ("s_nop 0\\n\\tv_mov_b32 %0, v3", [])])
def test_the_pattern_finds_written_registers(line, writes):
    assert WRITTEN.findall(line) == writes
