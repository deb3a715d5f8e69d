"""The paged cache's kernels start before the kernels in front of them are complete.  What they read and write of the call is visible, and free to
be written, behind their own wait only: checked in the source, since no run can show it."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "heddle_b200" / "csrc"


def _kernels():
    for name in ("kv_append_sm100.cu", "fa_paged_sm100.cuh", "fa_paged_tiles_sm100.cuh"):
        code = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
        for m in re.finditer(r"__global__[^{;]*?(\w+_kernel)\(", code):
            begin = code.index("{", m.end())
            depth, end = 0, begin
            while True:
                depth += {"{": 1, "}": -1}.get(code[end], 0)
                if depth == 0:
                    break
                end += 1
            yield m[1], code[begin:end]


@pytest.mark.parametrize("name,body", list(_kernels()), ids=lambda x: x if len(x) < 40 else "")
def test_waits_before_it_touches_memory(name, body):
    waits = [m.start() for m in re.finditer(r"\bgrid_wait\(\);", body)]
    assert len(waits) == 1 and not re.search(r"if \([^)]*\)\s*$", body[:waits[0]])
    before = body[:waits[0]]
    assert before.count("{") - before.count("}") == 1  # on the kernel's own level: every thread passes it
    assert "return" not in before
    # nothing of the call's memory in front of it: the cache, its tables, queries, outputs, workspace
    assert not re.search(r"kv_\w+\(|append_queries|paged_(?!tiles)\w+\(|p\.(q|o|k|v|lse|heads|parts|part_o|part_lse|cos|sin)\b", before.replace("p.tm_k", "").replace("p.tm_v", ""))


def test_all_kernels_are_looked_at():
    assert sorted(name for name, _ in _kernels()) == ["fa_paged_combine_kernel", "fa_paged_rows_kernel", "fa_paged_tiles_combine_kernel",
                                                      "fa_paged_tiles_kernel", "kv_append_kernel"]
