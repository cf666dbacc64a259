"""Runs the C++ tests of the group norm's plans (tests/cpp/plan_tests.cpp): host code, no GPU."""
import os
import subprocess

HERE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp")


def test_plans_hold_what_the_kernels_take_for_granted():
    path = os.path.join(HERE, "plan_tests")
    if not os.path.exists(path):
        subprocess.run(["make", "-C", HERE, "plan_tests"], check=True, capture_output=True)
    proc = subprocess.run([path], capture_output=True, text=True, timeout=120)
    tail = "\n".join(proc.stdout.splitlines()[-40:])
    assert proc.returncode == 0, f"plan_tests failed:\n{tail}\n{proc.stderr[-2000:]}"
    assert "3 case(s), 0 failure(s)" in proc.stdout
