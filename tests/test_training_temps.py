"""Temp of the operators of a training step: what is enough for a long call is enough for a shorter one, so that a program
may allocate once for its largest batch.  (The entry points compare temp_bytes with the size for their own arguments.)"""
import ctypes
import random

import pytest

from ilgpu_b200 import _native as N

L = N.lib()


def _bytes(function, *sizes):
    out = ctypes.c_int64(-1)
    assert getattr(L, function)(*sizes, ctypes.byref(out)) == N.OK, sizes
    return out.value


def _gradient(rows, width, tokens):
    return _bytes("b200alg_embedding_gradient_temp_bytes", rows, width, tokens)


def _growing(most, seed):
    """Lengths up to `most`, close together around powers of two and their small multiples."""
    rng = random.Random(seed)
    lengths = {0, 1, most} | {int(most ** rng.random()) for _ in range(2_000)}
    for k in range(31):
        for m in (1, 3, 111, 221, 222, 223):
            lengths |= {(m << k) + d for d in (-1, 0, 1)}
    return sorted(n for n in lengths if 0 <= n <= most)


@pytest.mark.parametrize("width", [1, 7, 8, 24, 64, 100, 768, 1_000, 1_024, 2_047, 2_048, 2_049, 4_096, 9_001, 65_536])
def test_more_tokens_never_need_less(width):
    sizes = [_gradient(32_000, width, n) for n in _growing((1 << 31) - 1, width)]
    assert sizes == sorted(sizes)


@pytest.mark.parametrize("tokens", [0, 1, 600, 1_025, 7_000, 8_192, 14_144, 16_384, 32_768, 300_000, 5_000_000, (1 << 31) - 1])
def test_wider_rows_never_need_less(tokens):
    sizes = [_gradient(32_000, width, tokens) for width in list(range(0, 4_200)) + [8_192, 20_001, 65_536, 1 << 20]]
    assert sizes == sorted(sizes)


def test_more_rows_never_need_less():
    sizes = [_gradient(rows, 512, 4_000) for rows in _growing((1 << 31) - 1, 3)]
    assert sizes == sorted(sizes)


def test_the_first_sizes_one_by_one():
    for width in (64, 2_048, 4_096):
        sizes = [_gradient(32_000, width, n) for n in range(0, 40_000)]
        assert sizes == sorted(sizes)


def test_norm_and_balance_loss():
    sizes = [_bytes("b200alg_gradient_norm_temp_bytes", n) for n in _growing((1 << 31) - 1, 4)]
    assert sizes == sorted(sizes)
    for experts in (1, 8, 60, 1_024):
        sizes = [_bytes("b200alg_balance_loss_temp_bytes", experts, n) for n in _growing((1 << 31) - 1, experts)]
        assert sizes == sorted(sizes)
    for tokens in (0, 40, 4_096, 100_000):
        sizes = [_bytes("b200alg_balance_loss_temp_bytes", experts, tokens) for experts in range(1, 1_025)]
        assert sizes == sorted(sizes)
