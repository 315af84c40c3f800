"""CPU test of the page table's checks of ragged appends and of lengths set for
many rows (csrc/page_table.cpp): the C++ unit test in tests/cpp_host is compiled
with g++ (no HIP) and run."""
from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


def test_ragged_host_checks(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    exe = tmp_path / "test_ragged_rows"
    cmd = [gxx, "-std=c++17", "-O1", "-Wall", "-Werror", f"-I{ROOT / 'include'}",
           f"-I{ROOT / 'streaming-attention_amd' / 'csrc'}", str(ROOT / "tests" / "cpp_host" / "test_ragged_rows.cpp"),
           str(ROOT / "streaming-attention_amd" / "csrc" / "page_table.cpp"), "-o", str(exe)]
    subprocess.run(cmd, check=True, capture_output=True, text=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True)
    assert res.returncode == 0, res.stdout + res.stderr
    assert "all checks passed" in res.stdout
