"""Runs the tests of the C++ mirror's wrappers for attention over selected blocks (tests/cpp/test_sparse.cpp)."""
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
BIN = os.path.join(HERE, "cpp", "_build", "test_sparse")


def _run(mode):
    if not os.path.exists(BIN):   # normally built by __graft_entry__.build()
        subprocess.run(["make", "-s", "-C", os.path.join(HERE, "cpp")], check=True)
    r = subprocess.run([BIN, mode], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "0 failure(s)" in r.stdout, r.stdout + r.stderr


def test_wrappers_cpu():
    _run("cpu")


@pytest.mark.gpu
def test_wrappers_gpu(dev):
    _run("gpu")
