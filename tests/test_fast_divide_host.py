"""Division by one product, which gives a group's row and column in the embedding's kernels (tests/cpp/fast_divide_test.cpp runs the
kernels' own code on the host).  No GPU."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)


def test_quotients(tmp_path):
    exe = str(tmp_path / "fast_divide_test")
    subprocess.check_call(["g++", "-std=c++17", "-O2", "-I", os.path.join(ROOT, "ilgpu_b200", "csrc"), os.path.join(HERE, "cpp", "fast_divide_test.cpp"), "-o", exe])
    run = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout + run.stderr
