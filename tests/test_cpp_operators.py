"""Runs the C++ tests of the training operators (tests/cpp/operator_tests.cpp) on the device."""
import os
import subprocess

import pytest

HERE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp")


@pytest.mark.gpu
def test_cpp_operators():
    path = os.path.join(HERE, "operator_tests")
    if not os.path.exists(path):
        subprocess.run(["make", "-C", HERE, "operator_tests"], check=True, capture_output=True)
    proc = subprocess.run([path], capture_output=True, text=True, timeout=120)
    tail = "\n".join(proc.stdout.splitlines()[-60:])
    assert proc.returncode == 0, f"operator_tests failed:\n{tail}\n{proc.stderr[-2000:]}"
    assert "4 case(s), 0 failure(s)" in proc.stdout
