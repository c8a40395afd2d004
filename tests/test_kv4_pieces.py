"""The join of cut units reads the partial rows of CTAs that the launch has,
whatever the entries hold that the kernel before left it (csrc/kv4_pieces.h, CPU only)."""

from __future__ import annotations

import re
import shutil
import subprocess
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent
CSRC = HERE.parent / "cuda-kv-persistence_b200" / "csrc"


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_pieces_are_the_launch_s(tmp_path):
    exe = tmp_path / "kv4_pieces_check"
    subprocess.run(["g++", "-O2", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", str(CSRC),
                    str(HERE / "kv4_pieces_check.cpp"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    assert "kv4 pieces ok" in out


def test_the_join_takes_its_pieces_from_there():
    text = (CSRC / "attn_kv4.cu").read_text()
    body = text[text.index("attn_kv4_join_units_kernel(const"):]
    body = body[: body.index("\n}\n")]
    assert re.findall(r"P\.ws_unit\[[^\]]*\]", re.sub(r"kv4_pieces\([^;]*\);", "", body)) == []
    assert body.count("kv4_pieces(") == 1
