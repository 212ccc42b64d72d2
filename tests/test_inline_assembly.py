"""Inline assembly of the kernels, as written.  m0 is reserved: the compiler lets no clobber list keep it, so assembly that
writes it has to leave what was there."""

from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "skmetal_amd" / "csrc"


def statements():
    for path in sorted(CSRC.iterdir()):
        for m in re.finditer(r"\basm\s*(?:volatile)?\s*\(", path.read_text()):
            text = path.read_text()[m.start():]
            yield path.name, text[: text.index(");") + 2]


def test_m0_is_left_as_it_was():
    found = 0
    for name, text in statements():
        code = "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', text.split(" : ")[0])).replace("\\n", "\n").replace("\\t", " ")
        lines = [ln.strip() for ln in code.split("\n") if ln.strip()]
        if not any(re.match(r"s_\w+ m0,", ln) for ln in lines):
            continue
        found += 1
        kept = re.fullmatch(r"s_mov_b32 (%\d+), m0", lines[0])
        assert kept and lines[-1] == f"s_mov_b32 m0, {kept[1]}", (name, lines)
        number = int(kept[1][1:])
        outputs = re.findall(r'"(=&?\w)"', text.split(" : ")[1])
        assert number < len(outputs) and outputs[number] == "=&s", (name, "kept in a register that no input shares")
    assert found == 2


@pytest.mark.parametrize("name", ["feed_kernels.hip"])
def test_statements_are_found(name):
    assert any(n == name for n, _ in statements())
