"""Runs the C++ host layer's attention test binary (tokspur-public_b200/native/tests/test_attention.cpp)."""
import os
import subprocess

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BIN = os.path.join(ROOT, "tokspur-public_b200", "native", "tests", "test_attention")


def test_attention_cpp_suite():
    if not os.path.exists(BIN):
        subprocess.run(["make", "-s", "-C", os.path.dirname(os.path.dirname(BIN))], check=True)
    r = subprocess.run([BIN], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "attention encode checks passed" in r.stdout
