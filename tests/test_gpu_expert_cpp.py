"""The C++ classes of the RMS norm, the router, the tokens' sort and the experts' products, end to end
(tests/cpp/expert_test.cpp)."""
import os
import subprocess

import pytest

from conftest import ROOT, log

pytestmark = pytest.mark.gpu

BIN = os.path.join(ROOT, "tests", "cpp", "expert_test")


def test_cpp_expert_program(gpu):
    assert os.path.exists(BIN), f"{BIN} missing: run __graft_entry__.build()"
    log("C++ expert program")
    r = subprocess.run([BIN], capture_output=True, text=True, timeout=90)
    print(r.stdout)
    lines = [ln for ln in r.stdout.splitlines() if ln.startswith(("ok ", "FAIL "))]
    assert r.returncode == 0, r.stdout + r.stderr
    assert len(lines) == 11 and all(ln.startswith("ok ") for ln in lines)
    assert "PASSED: 0 failure(s)" in r.stdout
