"""Runs the CPU tests of the launch plans of the operators over selected blocks (tests/cpp/test_sparse_plan.cpp)."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
BIN = os.path.join(HERE, "cpp", "_build", "test_sparse_plan")


def test_plans_fit():
    if not os.path.exists(BIN):   # normally built by __graft_entry__.build()
        subprocess.run(["make", "-s", "-C", os.path.join(HERE, "cpp")], check=True)
    r = subprocess.run([BIN], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and " 0 failure(s)" in r.stdout, r.stdout + r.stderr
