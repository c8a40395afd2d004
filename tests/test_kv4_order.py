"""The 4-bit cache's kernels are launched while what is before them in the
stream still runs: none of them may read device memory ahead of its wait."""

from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "cuda-kv-persistence_b200" / "csrc"
# what reads device memory: the helpers that look at starts, counts and the
# page map, and the pointers of the parameters
READS = re.compile(r"\b(unit_of|sequence|page_of|item_of|q_row|out_row|advance|Piece|add_partials|load16|fetch_rows)\s*[({]"
                   r"|\bP\.(ws_o|ws_ml|ws_unit|status)\b|(->|\.)(starts|counts|page_map|pages|q|out)\b|\*\s*reinterpret_cast")


def _kernels():
    for name in ("attn_kv4.cu", "attn_kv4_sm100.cu", "kv4_cache.cu"):
        text = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
        for m in re.finditer(r"__global__[^;{]*?(\w+_kernel)\s*\(", text):
            at = text.index("{", m.end())
            depth, end = 1, at + 1
            while depth:
                depth += {"{": 1, "}": -1}.get(text[end], 0)
                end += 1
            yield m.group(1), text[at:end]


def test_every_kernel_is_found():
    assert sorted(k for k, _ in _kernels()) == [
        "attn_kv4_join_kernel", "attn_kv4_join_units_kernel", "attn_kv4_rows_kernel", "attn_kv4_sm100_kernel",
        "kv4_read_kernel", "kv4_write_kernel"]


@pytest.mark.parametrize("name,body", list(_kernels()), ids=lambda x: x if x.endswith("_kernel") else "body")
def test_nothing_is_read_before_the_wait(name, body):
    before, wait, _ = body.partition("cudaGridDependencySynchronize()")
    assert wait
    early = READS.search(before.replace("*reinterpret_cast<RowsSmem<NB>*>(smem_raw)", ""))
    assert early is None, f"{name} reads {early.group(0)!r} before its wait"
