"""The batched-serving entry points without a device: structure layouts as a C compiler sees the header, and calls
without a context refused."""
from __future__ import annotations

import ctypes
import subprocess
from pathlib import Path

import pytest

REPO = Path(__file__).resolve().parent.parent

STRUCTS = {"PagedKV": ("lt_paged_kv", {"k": "dev_k", "v": "dev_v"}),
           "PagedAttnCfg": ("lt_paged_attn_cfg", {"slopes": "dev_slopes"}),
           "LogitRule": ("lt_logit_rule", {})}


def test_structures_match_the_header(pkg, tmp_path):
    lines = []
    for py, (c, names) in STRUCTS.items():
        lines.append(f'printf("{py} %zu\\n", sizeof({c}));')
        for f, _ in getattr(pkg, py)._fields_:
            lines.append(f'printf("{py}.{f} %zu\\n", offsetof({c}, {names.get(f, f)}));')
    src = tmp_path / "layout.c"
    src.write_text("#include <stdio.h>\n#include <stddef.h>\n#include \"llmtoy_cuda.h\"\nint main(void) {\n" +
                   "\n".join(lines) + "\nprintf(\"NO_MASK %u\\n\", LT_NO_MASK);\nreturn 0;\n}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", f"-I{REPO / 'include'}", str(src), "-o", str(exe)], check=True)
    got = dict(line.rsplit(" ", 1) for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    for py in STRUCTS:
        t = getattr(pkg, py)
        assert int(got[py]) == ctypes.sizeof(t)
        for f, _ in t._fields_:
            assert int(got[f"{py}.{f}"]) == getattr(t, f).offset, (py, f)
    assert int(got["NO_MASK"]) == pkg.NO_MASK


@pytest.mark.parametrize("name", ["lt_paged_append", "lt_paged_attn_decode", "lt_paged_attn_prompt", "lt_kv_evict",
                                  "lt_logits_process"])
def test_no_context_is_refused(pkg, name):
    fn = getattr(pkg.load_library(), name)
    args = [None if a is ctypes.c_void_p or hasattr(a, "contents") or issubclass(a, ctypes._Pointer) else 0 for a in fn.argtypes]
    assert fn(*args) == 1


def test_page_pool():
    import importlib
    serving = importlib.import_module("llmtoy-zig_b200.serving")
    p = serving.PagePool(5)
    a = p.take(3)
    assert len(set(a)) == 3
    with pytest.raises(MemoryError):
        p.take(3)
    p.give(a)
    assert sorted(p.take(5)) == list(range(5))
