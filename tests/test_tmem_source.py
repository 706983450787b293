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


def test_prompt_kernel_ends_after_its_copies_and_products():
    """A CTA that gave up on a wait, too, stays until its TMA copies and tensor-core products have ended: they write to
    its shared and tensor memory and arrive on its barriers.  A wait cannot be made to run out here without leaving
    copies behind, so the order is read from the source."""
    text = dict(sources())["lt_paged_prompt.cu"]
    kernel = text[text.index("void __launch_bounds__(kPpThreads, 1) k_paged_prompt("):text.index("kPpJoinRows")]
    end = kernel.rindex("tmem_dealloc(")
    # the copies: none after a wait ran out, and a bounded wait for the last of every stage behind the loop
    last = kernel.rindex("tma_load_4d(")
    assert "if (!__all_sync(0xffffffffu, wait(empty + st, (turn & 1) ^ 1))) continue;" in kernel[:last]
    assert re.search(r"for \(int i = 0; i < NS; i\+\+\)\s+if \(\(boxes_in >> i & 1u\) && !wait_always\(full \+ i,", kernel[last:end])
    # the products: one commit behind all of them, and a bounded wait for it
    last = max(kernel.rindex("umma_ts<"), kernel.rindex("qk(1,"), kernel.rindex("pv(tmem"))
    drain = re.search(r"umma_commit\(mma_end\);\s+__syncwarp\(\);\s+wait_always\(mma_end, 0\);", kernel[last:end])
    assert drain
    # both regardless of *dead
    always = kernel[kernel.index("auto wait_always"):kernel.index("auto wait =")]
    assert "mbar_wait_bounded(" in always and "if (!*dead)" not in always
