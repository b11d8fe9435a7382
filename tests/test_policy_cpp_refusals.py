"""CPU: what gym/hip_policy.h refuses from a C++ program (tests/cpp/hip_policy_refusals.cpp)."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BIN = os.path.join(ROOT, "tests", "cpp", "bin", "hip_policy_refusals")


def test_cpp_refusals():
    assert os.path.exists(BIN), "build tests/cpp first (python -c 'import __graft_entry__ as g; g.build()')"
    r = subprocess.run([BIN], capture_output=True, text=True, timeout=110)
    lines = r.stdout.strip().splitlines()
    assert r.returncode == 0 and len(lines) == 5 and all(line.startswith("ok ") for line in lines), (r.returncode, r.stdout, r.stderr[-2000:])
