"""Runs tests/cpp/training_step_test.cpp: the operators of a training step through include/ilgpu_algorithms.hpp."""
import os
import subprocess

import pytest

pytestmark = pytest.mark.gpu
CPP = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp")


def test_operators_through_the_cpp_mirror():
    exe = os.path.join(CPP, "training_step_test")
    if not os.path.exists(exe):
        subprocess.check_call(["make", "-C", CPP, "training_step_test"])
    run = subprocess.run([exe], capture_output=True, text=True, timeout=600)
    assert run.returncode == 0, run.stdout[-4000:] + run.stderr[-2000:]
    assert "0 failures" in run.stdout
