"""The norm of a list of views, and clipping by it, against 64 bits."""
import math

import pytest
import torch

import ilgpu_b200 as ib

from .training import NORM_BOUND, TYPES, assert_within, clipped, norm

pytestmark = pytest.mark.gpu

CHUNK = 8192
LISTS = {  # lengths of the views
    "one element": [1], "one": [1000], "empty ones": [0, 5, 0, 0, 7, 0], "chunk": [CHUNK - 1, CHUNK, CHUNK + 1, 2 * CHUNK, 3], "small ones": list(range(1, 200)),
    "large": [1_000_003, 17, 5_000_000], "many": [(i * 7919) % 400 for i in range(2_500)], "more than a launch lists": [3] * 1_025,
}


def _views(gen, lengths, kinds, packed, size=1.0):
    """Views of the given lengths, their types in turn; packed: one behind the other from an odd place on."""
    views = []
    for j, kind in enumerate(kinds):
        mine = lengths[j::len(kinds)]
        at = [1] if packed else [0]
        for n in mine:
            at.append(at[-1] + (n if packed else -(-n // 64) * 64))
        flat = (torch.randn(at[-1], generator=gen, device="cuda") * size).to(TYPES[kind])
        views += [flat[a:a + n] for a, n in zip(at, mine)]
    return views


def _temp(acc, views):
    temp = acc.Allocate1D(acc.ComputeGradientNormTempStorageSize(len(views)), torch.int32)
    temp.fill_(-1)
    return temp


def _norm(acc, views):
    out = torch.full((1,), -1.0, device="cuda")
    acc.CreateGradientNorm()(None, views, out, _temp(acc, views))
    return float(out)


@pytest.mark.parametrize("kinds", [["fp32"], ["bf16"], ["fp16"], ["bf16", "fp32"], ["fp16", "fp32", "bf16"]], ids="+".join)
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("name", LISTS)
def test_norm(accelerator, name, packed, kinds):
    views = _views(torch.Generator(device="cuda").manual_seed(len(name)), LISTS[name], kinds, packed)
    exact = norm(views)
    assert abs(_norm(accelerator, views) - exact) <= NORM_BOUND * exact


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("size", [1e-44, 1e-38, 1e-30, 1e-20, 1e-12, 1e15, 1e19, 1e25, 1e34])
def test_norm_where_squares_leave_the_range(accelerator, size, kind):
    gen = torch.Generator(device="cuda").manual_seed(3)
    views = _views(gen, [20_000, 3, 9_001], [kind], True, size)
    exact = norm(views)
    step = 2.0 ** -149  # of the result, where it is a subnormal
    assert abs(_norm(accelerator, views) - exact) <= NORM_BOUND * exact + step
    mixed = views + _views(gen, [50_000], [kind], False, size * 2.0 ** -12)  # beside values whose squares are smaller by 2^-24
    exact = norm(mixed)
    assert abs(_norm(accelerator, mixed) - exact) <= NORM_BOUND * exact + step


def test_norm_that_is_no_number(accelerator):
    views = [torch.ones(10_000, device="cuda"), torch.ones(77, dtype=torch.bfloat16, device="cuda")]
    assert _norm(accelerator, []) == 0.0
    assert _norm(accelerator, [torch.empty(0, device="cuda")]) == 0.0
    assert _norm(accelerator, [torch.zeros(30_000, device="cuda"), -torch.zeros(9, device="cuda")]) == 0.0
    views[0][9_999] = float("inf")
    assert _norm(accelerator, views) == math.inf
    views[1][76] = float("nan")
    assert math.isnan(_norm(accelerator, views))
    assert _norm(accelerator, [torch.full((4_000,), 3e38, device="cuda")]) == math.inf  # the norm itself is past the type


@pytest.mark.parametrize("types", ["fp32 fp32", "bf16 bf16", "fp32 bf16", "fp16 fp16", "bf16 fp32", "fp16 bf16", "fp32 fp16", "bf16 fp16", "fp16 fp32"])
@pytest.mark.parametrize("name", LISTS)
def test_clip(accelerator, name, types):
    source, target = types.split()
    gen = torch.Generator(device="cuda").manual_seed(len(name))
    for packed in (False, True):
        views = _views(gen, LISTS[name], [source], packed)
        before = [v.clone() for v in views]
        whole = norm(views)
        for max_norm in (whole / 3, whole * 2):
            out = torch.full((1,), -1.0, device="cuda")
            results = _views(gen, LISTS[name], [target], not packed if name == "chunk" else packed)
            accelerator.CreateGradientClip()(None, views, results, max_norm, out, _temp(accelerator, views))
            assert abs(float(out) - whole) <= NORM_BOUND * whole
            for v, b, r in list(zip(views, before, results))[:300]:
                assert torch.equal(v, b)
                assert_within(r, *clipped(b, float(out), max_norm, TYPES[target]))


@pytest.mark.parametrize("kinds", [["fp32"], ["bf16", "fp32"], ["fp16"]], ids="+".join)
def test_clip_in_place(accelerator, kinds):
    gen = torch.Generator(device="cuda").manual_seed(1)
    for lengths in ([5, 70_001, 0, 9], [(i * 31) % 300 for i in range(1_100)]):
        views = _views(gen, lengths, kinds, False)
        before = [v.clone() for v in views]
        out = torch.zeros(1, device="cuda")
        clip, temp = accelerator.CreateGradientClip(), _temp(accelerator, views)
        clip(None, views, None, 1e9, out, temp)
        assert all(torch.equal(v, b) for v, b in zip(views, before))
        clip(None, views, None, 0.5, out, temp)
        for v, b in zip(views, before):
            assert_within(v, *clipped(b, float(out), 0.5, v.dtype))
        clip(None, views, views, 0.0, out, temp)  # each output is its view
        assert not any(bool(v.any()) for v in views)


def test_some_views_in_place_and_some_not(accelerator):
    gen = torch.Generator(device="cuda").manual_seed(1)
    views = _views(gen, [70_001, 40_000, 9, 8_200, 100], ["bf16", "fp32"], True)
    before, out = [v.clone() for v in views], torch.zeros(1, device="cuda")
    for max_norm in (1e9, 2.0):
        outputs = [v if i % 2 else torch.full_like(v, 7.0, dtype=torch.float16) for i, v in enumerate(views)]
        accelerator.CreateGradientClip()(None, views, outputs, max_norm, out, _temp(accelerator, views))
        for v, b, o in zip(views, before, outputs):
            assert_within(o, *clipped(b, float(out), max_norm, o.dtype))
            assert v is o or torch.equal(v, b)


@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_a_norm_that_is_not_finite_changes_nothing(accelerator, bad):
    views = [torch.randn(9_000, device="cuda"), torch.randn(30, device="cuda").to(torch.bfloat16)]
    views[0][5] = bad
    before, out = [v.clone() for v in views], torch.zeros(1, device="cuda")
    accelerator.CreateGradientClip()(None, views, None, 1.0, out, _temp(accelerator, views))
    assert not math.isfinite(float(out))
    assert all(torch.equal(v.nan_to_num(7.0), b.nan_to_num(7.0)) for v, b in zip(views, before))
    results = [torch.empty_like(v, dtype=torch.float32) for v in views]
    accelerator.CreateGradientClip()(None, views, results, 1.0, out, _temp(accelerator, views))
    assert all(torch.equal(r.nan_to_num(7.0), b.float().nan_to_num(7.0)) for r, b in zip(results, before))


def test_scale_by_a_norm_that_is_given(accelerator):
    views = [torch.randn(300, 7, device="cuda"), torch.randn(40_000, device="cuda").to(torch.float16)]
    before, given = [v.clone() for v in views], torch.tensor([8.0], device="cuda")
    accelerator.CreateGradientScale()(None, views, None, 2.0, given)
    assert all(torch.equal(v, b * 0.25) for v, b in zip(views, before))  # a power of two: nothing is rounded
    accelerator.CreateGradientScale()(None, views, None, math.inf, given)
    assert all(torch.equal(v, b * 0.25) for v, b in zip(views, before))


def test_bits_do_not_change(accelerator):
    views = _views(torch.Generator(device="cuda").manual_seed(2), [3_000_001, 5, 77_777], ["bf16", "fp32"], True)
    first = _norm(accelerator, views)
    assert all(_norm(accelerator, views) == first for _ in range(5))


@pytest.mark.parametrize("count", [3, 65, 257, 1_100])
def test_captured_and_replayed(accelerator, count):
    """The lists of all table sizes, and of two launches, are the graph's own."""
    gen = torch.Generator(device="cuda").manual_seed(count)
    views = _views(gen, [(i * 37) % 500 for i in range(count)], ["fp32", "bf16"], True)
    results, out, temp = [torch.empty_like(v) for v in views], torch.zeros(1, device="cuda"), _temp(accelerator, views)
    clip = accelerator.CreateGradientClip()
    clip(None, views, results, 1.0, out, temp)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        clip(None, views, results, 1.0, out, temp)
        clip(None, views, results, 1.0, out, temp)
    for _ in range(3):
        for v in views:
            v.normal_(generator=gen)
        graph.replay()
        torch.cuda.synchronize()
        whole = norm(views)
        assert abs(float(out) - whole) <= NORM_BOUND * whole
        for v, r in list(zip(views, results))[::17]:
            assert_within(r, *clipped(v, float(out), 1.0, r.dtype))
    del graph


def test_a_view_past_32_bits_of_elements(accelerator):
    n = (1 << 32) + 77
    view = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    view[0], view[n - 1] = 3.0, 4.0
    assert _norm(accelerator, [view]) == 5.0
    out = torch.zeros(1, device="cuda")
    accelerator.CreateGradientClip()(None, [view], None, 2.5, out, _temp(accelerator, [view]))
    assert float(view[0]) == 1.5 and float(view[n - 1]) == 2.0 and not bool(view[1:n - 1].any())


def test_refusals(accelerator):
    clip, take, scale = accelerator.CreateGradientClip(), accelerator.CreateGradientNorm(), accelerator.CreateGradientScale()
    views, out = [torch.ones(4, 6, device="cuda"), torch.ones(3, device="cuda")], torch.zeros(1, device="cuda")
    temp = _temp(accelerator, views)
    for call, error in [
        (lambda: take(None, views[0], out, temp), ib.ArgumentNullException), (lambda: take(None, [None], out, temp), ib.ArgumentNullException),
        (lambda: take(None, [views[0].t()], out, temp), ib.NotSupportedException), (lambda: take(None, [views[0].double()], out, temp), ib.NotSupportedException),
        (lambda: take(None, [views[0].cpu()], out, temp), ib.InvalidOperationException), (lambda: take(None, views, out.double(), temp), ib.InvalidOperationException),
        (lambda: take(None, views, out[:0], temp), ib.ArgumentOutOfRangeException), (lambda: take(None, views, out, temp[:-1]), ib.ArgumentOutOfRangeException),
        (lambda: take(None, views, out, None), ib.ArgumentNullException), (lambda: clip(None, views, views[:1], 1.0, out, temp), ib.ArgumentOutOfRangeException),
        (lambda: clip(None, views, [views[1], views[0]], 1.0, out, temp), ib.ArgumentOutOfRangeException), (lambda: clip(None, views, None, -1.0, out, temp), ib.ArgumentOutOfRangeException),
        (lambda: clip(None, views, None, math.nan, out, temp), ib.ArgumentOutOfRangeException), (lambda: clip(None, views, None, 1.0, out, None), ib.ArgumentNullException),
        (lambda: scale(None, views, None, 1.0, None), ib.ArgumentNullException),
        (lambda: clip(None, views, [v.view(torch.int32) for v in views], 1.0, out, temp), ib.NotSupportedException),
    ]:
        with pytest.raises(error):
            call()
    assert all(bool((v == 1.0).all()) for v in views)
