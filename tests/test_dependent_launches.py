"""A kernel that may start while the one before it still runs finds what that one, and all before it, wrote only behind its
wait: each kernel of the operators of a training step waits on every path, in front of its first access to memory."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ilgpu_b200", "csrc")
WAIT = "grid_dependency_wait();"


def _body(text, at):
    """The braces' content from the first one behind `at` on."""
    begin = text.index("{", at)
    depth = 0
    for i in range(begin, len(text)):
        depth += (text[i] == "{") - (text[i] == "}")
        if not depth:
            return text[begin + 1:i]
    raise AssertionError("unbalanced braces")


def _source(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def _kernels(text):
    for match in re.finditer(r"__global__ void\s+(?:__launch_bounds__\((?:[^()]|\([^()]*\))*\)\s*)?(\w+)\(", text):
        yield match.group(1), _body(text, match.end())


SOURCES = ["embedding.cu", "gradient_norm.cu", "balance_loss.cu"]


def test_the_kernels_are_found():
    assert {name for source in SOURCES for name, _ in _kernels(_source(source))} >= {
        "lookup_kernel", "gradient_sum_kernel", "gradient_join_kernel", "gradient_few_kernel", "norm_partial_kernel", "scale_kernel", "balance_kernel",
        "balance_finish_kernel", "balance_gradient_kernel"}


@pytest.mark.parametrize("source", SOURCES)
def test_no_kernel_goes_without_its_wait(source):
    text = _source(source)
    for name, body in _kernels(text):
        if WAIT not in body:  # in the function that does the kernel's work
            called = [_body(text, m.start()) for m in re.finditer(r"__device__ [^;{]*\b(\w+)\([^;{]*\{", text) if re.search(rf"\b{m.group(1)}\s*[<(]", body)]
            assert any(WAIT in function for function in called), f"{name} does not wait"
            continue
        assert not re.search(r"\bif\s*\([^;{]*\)\s*" + re.escape(WAIT), body), f"{name} waits only at times"
        # where a block of statements returns, it, or what comes in front of it, has waited
        for match in re.finditer(r"\breturn\b", body):
            assert WAIT in body[:match.start()], f"{name} returns without a wait"
