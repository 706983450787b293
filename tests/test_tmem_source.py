"""Loads from tensor memory: the registers of a tcgen05.ld are undefined until tcgen05.wait::ld, and a compiler may
move a use of them before a wait that does not name them.  No output shows that with a compiler that does not, so the
sources are checked: a load and its wait are one statement, or the wait names what was loaded."""
from __future__ import annotations

import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "llmtoy-zig_b200" / "csrc"


def sources():
    for p in sorted([*CSRC.glob("*.cu"), *CSRC.glob("*.cuh")]):
        yield p.name, re.sub(r"//[^\n]*", "", p.read_text())


def test_every_wait_names_what_it_waits_for():
    for name, text in sources():
        assert not re.search(r"\btmem_wait_ld\s*\(\s*\)", text), name
        # the wait itself stands in its helper and in single-column loads, nowhere else
        for m in re.finditer(r"tcgen05\.wait::ld", text):
            stmt = text[text.rfind("asm", 0, m.start()):text.index(";\n", text.index(");", m.start()))]
            helper = text[:m.start()].rstrip().endswith('asm volatile("') and name == "lt_umma.cuh"
            assert helper or "tcgen05.ld." in stmt, name


def test_scalar_loads_carry_their_wait():
    """A value returned by a function cannot be named by a wait behind it."""
    found = 0
    for name, text in sources():
        for m in re.finditer(r'"tcgen05\.ld\.[^"]*\.x1\.b32[^"]*"', text):
            found += 1
            assert "tcgen05.wait::ld" in m.group(0), name
    assert found
