"""GPU: gym/hip_policy.h from a C++ program (tests/cpp/hip_policy_demo.cpp), without Python between."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BIN = os.path.join(ROOT, "tests", "cpp", "bin", "hip_policy_demo")


@pytest.mark.gpu
def test_cpp_trainer_calls():
    assert os.path.exists(BIN), "build tests/cpp first (python -c 'import __graft_entry__ as g; g.build()')"
    r = subprocess.run([BIN], capture_output=True, text=True, timeout=110)
    lines = r.stdout.strip().splitlines()
    assert r.returncode == 0 and len(lines) == 13 and all(line.startswith("ok ") for line in lines), (r.returncode, r.stdout, r.stderr[-2000:])
