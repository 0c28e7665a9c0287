"""Rules of the kernels' waits that can be read from their sources (a wait that
breaks one could hang a GPU, so none is tried on one)."""
from __future__ import annotations

from pathlib import Path
import re

import pytest

SOURCES = sorted((Path(__file__).resolve().parents[1] / "graph_rewrite_system_b200" / "csrc")
                 .glob("*.cu*"))


def _condition(text: str, at: int) -> str:
    """The parenthesised text that opens at `at`."""
    depth = 0
    for i in range(at, len(text)):
        depth += {"(": 1, ")": -1}.get(text[i], 0)
        if not depth:
            return text[at:i + 1]
    raise AssertionError("unbalanced")


def _loose_reads(text: str) -> list[str]:
    """Loop conditions that read a volatile flag lane by lane: where the loop
    makes a collective wait, lanes that saw different values would part."""
    flags = re.findall(r"\bvolatile\s+\w+\s*\*\s*(\w+)", text)
    bad = []
    for loop in re.finditer(r"\bwhile\s*\(", text):
        condition = _condition(text, loop.end() - 1)
        body = text[loop.end() - 1:loop.end() + len(condition) + 300]
        if not re.search(r"_sync\(|mbar_wait_warp\(", body):
            continue
        voted = re.sub(r"__(any|all)_sync\([^()]*\)", "", condition)
        bad += [condition for flag in flags if re.search(rf"\*\s*{flag}\b", voted)]
    return bad


@pytest.mark.parametrize("source", SOURCES, ids=lambda p: p.name)
def test_loops_around_collective_waits_leave_as_a_warp(source):
    assert not _loose_reads(source.read_text())


def test_the_rule_sees_both_forms():
    head = "volatile int* flag = &failed;\n"
    assert _loose_reads(head + "while (!ok && !*flag) ok = mbar_wait_warp(&bar, 0);")
    assert not _loose_reads(
        head + "while (!ok && !__any_sync(0xffffffffu, *flag)) ok = mbar_wait_warp(&bar, 0);")
