"""GPU: host memory that runs out inside a decode or a fused step is an error
(tests/cpp/test_host_memory.cpp, one PASS/FAIL line per check)."""
from __future__ import annotations

import subprocess
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

EXE = Path(__file__).resolve().parent / "cpp" / "bin" / "test_host_memory"


def test_host_memory_that_runs_out_is_an_error():
    assert EXE.exists(), "C++ driver missing: python streaming-attention_amd/build.py --tests"
    r = subprocess.run([str(EXE)], capture_output=True, text=True, timeout=100)
    failed = [line for line in r.stdout.splitlines() if line.startswith("FAIL")]
    assert r.returncode == 0 and not failed, "\n".join(failed) + r.stderr
    assert r.stdout.count("PASS") == 3 * 13
