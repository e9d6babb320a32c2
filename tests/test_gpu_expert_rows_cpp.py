"""Rows that are only copied, through the C++ class of the tokens' sort (tests/cpp/expert_rows_test.cpp)."""
import os
import subprocess

import pytest

from conftest import ROOT, log

pytestmark = pytest.mark.gpu

BIN = os.path.join(ROOT, "tests", "cpp", "expert_rows_test")


def test_cpp_expert_rows_program(gpu):
    assert os.path.exists(BIN), f"{BIN} missing: run __graft_entry__.build()"
    log("C++ program of copied rows")
    r = subprocess.run([BIN], capture_output=True, text=True, timeout=90)
    print(r.stdout)
    lines = [ln for ln in r.stdout.splitlines() if ln.startswith(("ok ", "FAIL "))]
    assert r.returncode == 0, r.stdout + r.stderr
    assert len(lines) == 6 and all(ln.startswith("ok ") for ln in lines)
    assert "PASSED: 0 failure(s)" in r.stdout
