"""What the operators of a training step refuse, through the C ABI: every refusal comes back before any CUDA call, so
this runs without a GPU.  Pointers are only checked for null and alignment."""
import ctypes

import pytest

from ilgpu_b200 import _native as N

L = N.lib()
P = ctypes.c_void_p(4096)          # aligned
ODD = ctypes.c_void_p(4097)        # aligned to nothing
BIG = 1 << 40
INVALID, UNSUPPORTED, SMALL, MISALIGNED, LARGE = N.INVALID_ARGUMENT, N.UNSUPPORTED, N.TEMP_TOO_SMALL, N.MISALIGNED, N.TOO_LARGE


def _call(function, defaults, **changed):
    assert set(changed) <= set(defaults)
    return getattr(L, function)(*(defaults | changed).values())


EMBED = dict(stream=None, table=P, rows=10, width=16, row_stride=16, dtype=N.BF16, tokens=P, n=4, token_stride=1, token_dtype=N.I32, scale=1.0,
             out=P, out_stride=16, out_dtype=N.F32)


@pytest.mark.parametrize("changed, status", [
    (dict(rows=-1), INVALID), (dict(width=-1), INVALID), (dict(n=-1), INVALID), (dict(token_stride=0), INVALID), (dict(row_stride=15), INVALID),
    (dict(out_stride=-16), INVALID), (dict(row_stride=1 << 60), INVALID), (dict(table=None), INVALID), (dict(tokens=None), INVALID),
    (dict(out=None), INVALID), (dict(dtype=N.F64), UNSUPPORTED), (dict(dtype=N.I32), UNSUPPORTED), (dict(out_dtype=99), UNSUPPORTED),
    (dict(token_dtype=N.U32), UNSUPPORTED), (dict(token_dtype=N.F32), UNSUPPORTED), (dict(n=1 << 31), LARGE), (dict(rows=1 << 31), LARGE),
    (dict(table=ODD), MISALIGNED), (dict(out=ODD), MISALIGNED), (dict(tokens=ODD), MISALIGNED), (dict(tokens=ctypes.c_void_p(4100), token_dtype=N.I64), MISALIGNED),
])
def test_embedding(changed, status):
    assert _call("b200alg_embedding", EMBED, **changed) == status


def test_nothing_to_look_up():
    assert _call("b200alg_embedding", EMBED, n=0, tokens=None, out=None) == N.OK
    assert _call("b200alg_embedding", EMBED, width=0, table=None, out=None, row_stride=0, out_stride=0) == N.OK


GRADIENT = dict(stream=None, tokens=P, n=4, token_stride=1, token_dtype=N.I64, upstream=P, upstream_stride=16, upstream_dtype=N.F16, scale=1.0,
                gradient=P, rows=10, width=16, row_stride=16, dtype=N.F32, accumulate=0, temp=P, temp_bytes=BIG)


@pytest.mark.parametrize("changed, status", [
    (dict(n=-1), INVALID), (dict(rows=-1), INVALID), (dict(width=-1), INVALID), (dict(token_stride=-1), INVALID), (dict(upstream_stride=8), INVALID),
    (dict(row_stride=15), INVALID), (dict(tokens=None), INVALID), (dict(upstream=None), INVALID), (dict(gradient=None), INVALID),
    (dict(temp=None), INVALID), (dict(upstream_dtype=N.F64), UNSUPPORTED), (dict(dtype=N.U16), UNSUPPORTED), (dict(token_dtype=N.U64), UNSUPPORTED),
    (dict(n=1 << 31), LARGE), (dict(rows=1 << 31, row_stride=16), LARGE), (dict(temp=ctypes.c_void_p(4096 + 128)), MISALIGNED),
    (dict(gradient=ODD), MISALIGNED), (dict(upstream=ODD), MISALIGNED), (dict(tokens=ctypes.c_void_p(4100)), MISALIGNED), (dict(temp_bytes=0), SMALL),
])
def test_embedding_gradient(changed, status):
    assert _call("b200alg_embedding_gradient", GRADIENT, **changed) == status


def _need(function, *arguments):
    out = ctypes.c_int64(-1)
    return getattr(L, function)(*arguments, ctypes.byref(out)), out.value


def test_embedding_gradient_temp():
    status, need = _need("b200alg_embedding_gradient_temp_bytes", 10, 16, 4)
    assert status == N.OK and need % 256 == 0
    assert _call("b200alg_embedding_gradient", GRADIENT, temp_bytes=need - 1) == SMALL
    assert _need("b200alg_embedding_gradient_temp_bytes", 10, 16, -1)[0] == INVALID
    assert _need("b200alg_embedding_gradient_temp_bytes", 10, 16, 1 << 31)[0] == LARGE
    assert L.b200alg_embedding_gradient_temp_bytes(10, 16, 4, None) == INVALID
    # sizes past 32 bits: shares of a long input over a wide table
    status, need = _need("b200alg_embedding_gradient_temp_bytes", 128_000, 65_536, (1 << 31) - 1)
    assert status == N.OK and need > 1 << 32


def _lists(pointers, lengths, types):
    return ((ctypes.c_void_p * len(pointers))(*[p.value if p else None for p in pointers]), (ctypes.c_int64 * len(lengths))(*lengths),
            (ctypes.c_int * len(types))(*types))


VIEWS = _lists([P, P], [5, 7], [N.F32, N.BF16])
NORM = dict(stream=None, views=VIEWS[0], lengths=VIEWS[1], dtypes=VIEWS[2], count=2, norm=P, temp=P, temp_bytes=BIG)
CLIP = dict(stream=None, views=VIEWS[0], outputs=_lists([ctypes.c_void_p(8192)] * 2, [], [])[0], lengths=VIEWS[1], dtypes=VIEWS[2], out_dtypes=VIEWS[2],
            count=2, max_norm=1.0, norm=P, temp=P, temp_bytes=BIG)
SCALE = {k: CLIP[k] for k in ("stream", "views", "outputs", "lengths", "dtypes", "out_dtypes", "count", "norm", "max_norm")}


@pytest.mark.parametrize("function, defaults", [("b200alg_gradient_norm", NORM), ("b200alg_gradient_clip", CLIP), ("b200alg_gradient_scale", SCALE)])
@pytest.mark.parametrize("changed, status", [
    (dict(count=-1), INVALID), (dict(views=None), INVALID), (dict(lengths=None), INVALID), (dict(dtypes=None), INVALID), (dict(norm=None), INVALID),
    (dict(norm=ODD), MISALIGNED), (dict(views=_lists([P, None], [], [])[0]), INVALID), (dict(views=_lists([P, ODD], [], [])[0]), MISALIGNED),
    (dict(lengths=_lists([], [5, -1], [])[1]), INVALID), (dict(lengths=_lists([], [1 << 37, (1 << 37) + 1], [])[1]), LARGE),
    (dict(dtypes=_lists([], [], [N.F32, N.F64])[2]), UNSUPPORTED), (dict(dtypes=_lists([], [], [N.I32, N.F32])[2]), UNSUPPORTED),
])
def test_lists_of_views(function, defaults, changed, status):
    assert _call(function, defaults, **changed) == status


@pytest.mark.parametrize("function, defaults", [("b200alg_gradient_clip", CLIP), ("b200alg_gradient_scale", SCALE)])
@pytest.mark.parametrize("changed, status", [
    (dict(max_norm=-1.0), INVALID), (dict(max_norm=float("nan")), INVALID), (dict(outputs=_lists([P, None], [], [])[0]), INVALID),
    (dict(outputs=_lists([P, ODD], [], [])[0]), MISALIGNED), (dict(out_dtypes=_lists([], [], [N.F32, N.I8])[2]), UNSUPPORTED),
    # in place the type cannot change
    (dict(outputs=None, out_dtypes=_lists([], [], [N.F32, N.F32])[2]), INVALID), (dict(outputs=VIEWS[0], out_dtypes=_lists([], [], [N.F16, N.BF16])[2]), INVALID),
])
def test_clipping(function, defaults, changed, status):
    assert _call(function, defaults, **changed) == status


def test_norm_temp():
    for count in (0, 1, 5_000):
        status, need = _need("b200alg_gradient_norm_temp_bytes", count)
        assert status == N.OK and need % 256 == 0
    assert _need("b200alg_gradient_norm_temp_bytes", -1)[0] == INVALID
    assert _call("b200alg_gradient_norm", NORM, temp_bytes=255) == SMALL
    assert _call("b200alg_gradient_clip", CLIP, temp_bytes=255) == SMALL
    assert _call("b200alg_gradient_norm", NORM, temp=ctypes.c_void_p(4096 + 64)) == MISALIGNED
    assert _call("b200alg_gradient_clip", CLIP, temp=None) == INVALID


BALANCE = dict(stream=None, logits=P, tokens=4, experts=8, logits_stride=8, dtype=N.F32, chosen=P, choices=2, chosen_stride=2, chosen_dtype=N.I64,
               mask=None, coefficient=0.01, loss=P, counts=P, probabilities=P, temp=P, temp_bytes=BIG)
BALANCE_GRADIENT = dict(stream=None, logits=P, tokens=4, experts=8, logits_stride=8, dtype=N.F32, mask=None, counts=P, choices=2, coefficient=0.01,
                        loss_gradient=P, gradient=P, gradient_stride=8, accumulate=0)


@pytest.mark.parametrize("function, defaults", [("b200alg_balance_loss", BALANCE), ("b200alg_balance_loss_gradient", BALANCE_GRADIENT)])
@pytest.mark.parametrize("changed, status", [
    (dict(tokens=-1), INVALID), (dict(experts=0), INVALID), (dict(choices=0), INVALID), (dict(logits_stride=7), INVALID), (dict(logits=None), INVALID),
    (dict(counts=None), INVALID), (dict(coefficient=float("inf")), INVALID), (dict(coefficient=float("nan")), INVALID), (dict(dtype=N.F64), UNSUPPORTED),
    (dict(experts=1025, logits_stride=1025), UNSUPPORTED), (dict(tokens=(1 << 30) + 1, choices=2), LARGE), (dict(logits=ODD), MISALIGNED),
    (dict(counts=ODD), MISALIGNED),
])
def test_balance_loss_and_gradient(function, defaults, changed, status):
    if "gradient_stride" in defaults and "experts" in changed:
        changed = changed | {"gradient_stride": max(8, changed["experts"])}
    assert _call(function, defaults, **changed) == status


@pytest.mark.parametrize("changed, status", [
    (dict(chosen=None), INVALID), (dict(loss=None), INVALID), (dict(probabilities=None), INVALID), (dict(temp=None), INVALID), (dict(chosen_stride=1), INVALID),
    (dict(chosen_dtype=N.U32), UNSUPPORTED), (dict(chosen_dtype=N.F32), UNSUPPORTED), (dict(temp_bytes=255), SMALL), (dict(chosen=ctypes.c_void_p(4100)), MISALIGNED),
    (dict(loss=ODD), MISALIGNED), (dict(probabilities=ODD), MISALIGNED), (dict(temp=ctypes.c_void_p(4096 + 64)), MISALIGNED),
])
def test_balance_loss(changed, status):
    assert _call("b200alg_balance_loss", BALANCE, **changed) == status


@pytest.mark.parametrize("changed, status", [
    (dict(loss_gradient=None), INVALID), (dict(gradient=None), INVALID), (dict(gradient_stride=7), INVALID), (dict(gradient=ODD), MISALIGNED),
    (dict(loss_gradient=ODD), MISALIGNED),
])
def test_balance_loss_gradient(changed, status):
    assert _call("b200alg_balance_loss_gradient", BALANCE_GRADIENT, **changed) == status


def test_balance_temp():
    status, need = _need("b200alg_balance_loss_temp_bytes", 8, 4)
    assert status == N.OK and need % 256 == 0
    assert _call("b200alg_balance_loss", BALANCE, temp_bytes=need - 1) == SMALL
    assert _need("b200alg_balance_loss_temp_bytes", 0, 4)[0] == INVALID
    assert _need("b200alg_balance_loss_temp_bytes", 2_000, 4)[0] == UNSUPPORTED
    assert _call("b200alg_balance_loss_gradient", BALANCE_GRADIENT, tokens=0, logits=None, gradient=None) == N.OK


def test_the_other_entry_points_know_no_bf16():
    """The type is one of these operators' alone."""
    assert _need("b200alg_radix_sort_temp_bytes", N.BF16, 10, 0)[0] == UNSUPPORTED
    assert _need("b200alg_scan_temp_bytes", N.BF16, 10)[0] == UNSUPPORTED
    assert L.b200alg_reduce(None, P, 1, 10, N.BF16, N.ADD, P) == UNSUPPORTED
    assert _need("b200alg_unique_temp_bytes", N.BF16, 10)[0] == UNSUPPORTED
