"""The balance loss of a router with the counts per expert, and its gradient, against 64 bits and against differences."""
import math

import pytest
import torch

import ilgpu_b200 as ib

from .training import TYPES, Balance, assert_within

pytestmark = pytest.mark.gpu
COEFFICIENT = 0.01


def _run(acc, logits, chosen, mask=None, coefficient=COEFFICIENT):
    tokens, experts = logits.shape
    loss, counts, p = torch.full((1,), -1.0, device="cuda"), torch.full((experts + 3,), -7, dtype=torch.int32, device="cuda"), torch.full((experts + 2,), -1.0, device="cuda")
    temp = acc.Allocate1D(acc.ComputeBalanceLossTempStorageSize(experts, tokens), torch.int32)
    temp.fill_(-1)
    acc.CreateBalanceLoss(coefficient)(None, logits, chosen, mask, loss, counts, p, temp)
    assert bool((counts[experts + 1:] == -7).all()) and bool((p[experts:] == -1.0).all())
    return loss, counts[:experts + 1], p[:experts]


def _check(acc, logits, chosen, mask=None):
    b = Balance(logits, chosen, mask, COEFFICIENT)
    loss, counts, p = _run(acc, logits, chosen, mask)
    assert counts.tolist() == b.counts.tolist() + [b.number]
    value, bound, mean, off = b.loss()
    assert_within(p, mean, off)
    assert_within(loss, value, bound)
    upstream = torch.tensor([3.0 * max(1, b.number)], device="cuda")
    for base in (None, torch.randn(logits.shape, device="cuda").to(logits.dtype)):
        gradient = torch.full(logits.shape, float("nan"), dtype=logits.dtype, device="cuda") if base is None else base.clone()
        acc.CreateBalanceLossGradient(COEFFICIENT, chosen.shape[1], base is not None)(None, logits, mask, counts, upstream, gradient)
        assert_within(gradient, *b.gradient(float(upstream), logits.dtype, base=base))
        if base is not None:
            assert torch.equal(gradient[~b.valid.cuda()], base[~b.valid.cuda()])


def _router(gen, tokens, experts, choices, kind, ids, spread=2.0):
    logits = (torch.randn(tokens, experts, generator=gen, device="cuda") * spread).to(TYPES[kind])
    return logits, torch.randint(0, experts, (tokens, choices), generator=gen, device="cuda").to(ids)


@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("tokens, experts, choices", [
    (1, 1, 1), (1, 8, 2), (2, 3, 1), (31, 4, 4), (64, 8, 2), (65, 16, 3), (100, 24, 2), (1_000, 60, 4), (515, 61, 5), (2_000, 64, 8), (777, 128, 1), (130, 130, 2),
    (3_001, 160, 6), (500, 256, 8), (129, 257, 8), (70, 320, 2), (90, 512, 4), (40, 513, 3), (33, 768, 8), (20, 1_000, 2), (50, 1_023, 16), (48, 1_024, 1),
    (500, 21, 2), (501, 30, 3), (300, 38, 4), (301, 44, 2), (302, 62, 6), (200, 70, 2), (201, 93, 4), (150, 101, 2), (151, 122, 8), (70, 252, 2), (71, 258, 2), (60, 514, 2),
    (40, 1_018, 3), (41, 1_012, 3), (1, 1_024, 2), (4, 1_024, 8), (3, 1_023, 2), (4, 1_000, 1)])
def test_loss_and_gradient(accelerator, tokens, experts, choices, kind):
    gen = torch.Generator(device="cuda").manual_seed(tokens + experts)
    logits, chosen = _router(gen, tokens, experts, choices, kind, torch.int64 if tokens % 2 else torch.int32)
    _check(accelerator, logits, chosen)
    mask = torch.rand(tokens, generator=gen, device="cuda") < 0.6
    logits[~mask], chosen[~mask] = float("nan"), 1 << 30  # what the mask leaves out is not read
    _check(accelerator, logits, chosen, mask)
    _check(accelerator, logits, chosen, mask.to(torch.uint8) * 200)
    _check(accelerator, logits, chosen, torch.zeros_like(mask))  # no token counts


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_many_tokens(accelerator, kind):
    gen = torch.Generator(device="cuda").manual_seed(1)
    logits, chosen = _router(gen, 100_003, 40, 3, kind, torch.int32)
    _check(accelerator, logits, chosen)
    _check(accelerator, logits, chosen, torch.rand(100_003, generator=gen, device="cuda") < 0.5)


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("experts, stride, offset", [(8, 9, 0), (64, 72, 0), (64, 64, 1), (60, 64, 4), (7, 16, 3), (128, 130, 2), (256, 264, 8)])
def test_strided_views(accelerator, kind, experts, stride, offset):
    gen = torch.Generator(device="cuda").manual_seed(experts)
    tokens, choices = 333, 3
    flat = torch.full((offset + tokens * stride,), float("nan"), device="cuda").to(TYPES[kind])
    logits = flat[offset:].as_strided((tokens, experts), (stride, 1))
    logits.copy_(torch.randn(tokens, experts, generator=gen, device="cuda"))
    chosen = torch.full((tokens, choices + 4), 5, device="cuda")[:, :choices]
    chosen.copy_(torch.randint(0, experts, (tokens, choices), generator=gen, device="cuda"))
    _check(accelerator, logits, chosen)
    b = Balance(logits, chosen, None, COEFFICIENT)
    out = torch.full_like(flat, 9.0)
    gradient = out[offset:].as_strided((tokens, experts), (stride, 1))
    _, counts, _ = _run(accelerator, logits, chosen)
    accelerator.CreateBalanceLossGradient(COEFFICIENT, choices)(None, logits, None, counts, torch.tensor([500.0], device="cuda"), gradient)
    assert_within(gradient, *b.gradient(500.0, logits.dtype))
    gradient.fill_(9.0)
    assert bool((out == 9.0).all())


def test_rows_of_extremes(accelerator):
    gen = torch.Generator(device="cuda").manual_seed(4)
    for kind in ("fp32", "bf16", "fp16"):
        logits, chosen = _router(gen, 64, 24, 2, kind, torch.int64)
        info = torch.finfo(logits.dtype)
        logits[3] = -math.inf                      # no expert may be chosen: p = 0
        logits[4, ::2] = -math.inf                 # some may not
        logits[5] = info.min                       # all at the type's lowest value: uniform
        logits[6], logits[6, 1] = info.min, 0.0
        logits[7], logits[7, 5] = 0.0, info.max    # one takes all
        logits[8] = info.max
        logits[9], logits[9, 0] = -math.inf, info.min
        _check(accelerator, logits, chosen)


@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_what_is_not_a_number_comes_through(accelerator, bad):
    gen = torch.Generator(device="cuda").manual_seed(4)
    logits, chosen = _router(gen, 70, 12, 2, "fp32", torch.int64)
    logits[40, 3] = bad
    loss, counts, p = _run(accelerator, logits, chosen)
    assert math.isnan(float(loss)) and bool(torch.isnan(p).all()) and int(counts.sum()) == 70 * 2 + 70
    gradient = torch.zeros_like(logits)
    accelerator.CreateBalanceLossGradient(COEFFICIENT, 2)(None, logits, None, counts, torch.ones(1, device="cuda"), gradient)
    nan = torch.isnan(gradient)
    assert bool(nan[40].all()) and int(nan.sum()) == 12


def test_choices_that_are_none(accelerator):
    """Indices outside the experts, as a router gives them for tokens that it drops, are not counted."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    for ids in (torch.int32, torch.int64):
        logits, chosen = _router(gen, 200, 10, 3, "fp32", ids)
        chosen[::3, 0], chosen[1::3, 1], chosen[5] = -1, 10, torch.iinfo(ids).max
        chosen[6] = torch.iinfo(ids).min
        if ids == torch.int64:
            chosen[7] = (1 << 32) + 1
        _check(accelerator, logits, chosen)


def test_no_tokens(accelerator):
    loss, counts, p = _run(accelerator, torch.empty(0, 9, device="cuda"), torch.empty(0, 2, dtype=torch.int64, device="cuda"))
    assert float(loss) == 0.0 and not bool(counts.any()) and not bool(p.any())
    empty = torch.empty(0, 9, device="cuda")
    accelerator.CreateBalanceLossGradient(COEFFICIENT, 2)(None, empty, None, counts, torch.ones(1, device="cuda"), empty)


def test_gradient_against_differences(accelerator):
    """The loss of the definition in 64 bits along random directions: a central difference is off by h^2 times the third derivative."""
    gen = torch.Generator(device="cuda").manual_seed(8)
    logits, chosen = _router(gen, 50, 12, 2, "fp32", torch.int64)
    _, counts, _ = _run(accelerator, logits, chosen, coefficient=1.0)
    gradient = torch.empty_like(logits)
    accelerator.CreateBalanceLossGradient(1.0, 2)(None, logits, None, counts, torch.ones(1, device="cuda"), gradient)
    for _ in range(5):
        d = torch.randn(logits.shape, generator=gen, device="cuda").double()
        h = 1e-4
        up, down = (float(Balance(logits.double() + s * h * d, chosen, None, 1.0).loss()[0]) for s in (1, -1))
        slope = float((gradient.double() * d).sum())
        # the loss is an average of softmaxes times weights of at most E: its third derivative along d is below E max|d|^3, the difference's
        # rounding 1e-15 / h, the gradient's own bound 1e-5 of its size
        assert abs((up - down) / (2 * h) - slope) <= h * h * 12 * float(d.abs().max()) ** 3 + 1e-11 + 1e-5 * float((gradient.double() * d).abs().sum())


@pytest.mark.parametrize("tokens, experts, stride", [(1, 1, 1), (300, 8, 8), (123, 60, 60), (77, 61, 64), (40, 300, 301), (9, 1_024, 1_024)])
def test_experts_chosen_alike(accelerator, tokens, experts, stride):
    """Where every expert is chosen as often, nothing is to be learnt: the gradient is zero, not what rounding leaves of it."""
    gen = torch.Generator(device="cuda").manual_seed(10)
    logits = torch.randn(tokens, stride, generator=gen, device="cuda")[:, :experts]
    chosen = torch.arange(experts, device="cuda").expand(tokens, experts).contiguous()
    _, counts, _ = _run(accelerator, logits, chosen)
    assert counts.tolist() == [tokens] * (experts + 1)
    gradient = torch.full((tokens, experts), math.nan, device="cuda")
    accelerator.CreateBalanceLossGradient(1.0, experts)(None, logits, None, counts, torch.full((1,), 1e6, device="cuda"), gradient)
    assert not bool(gradient.any())


def test_counts_of_all_ranks(accelerator):
    """Counts and tokens that were summed over ranks."""
    gen = torch.Generator(device="cuda").manual_seed(9)
    logits, chosen = _router(gen, 300, 20, 2, "bf16", torch.int64)
    counts = torch.randint(0, 5_000, (21,), generator=gen, device="cuda").to(torch.int32)
    counts[20] = 2_400
    gradient = torch.empty_like(logits)
    accelerator.CreateBalanceLossGradient(COEFFICIENT, 2)(None, logits, None, counts, torch.tensor([2.0], device="cuda"), gradient)
    assert_within(gradient, *Balance(logits, chosen, None, COEFFICIENT).gradient(2.0, logits.dtype, counts, 2_400))


def test_bits_do_not_change(accelerator):
    logits, chosen = _router(torch.Generator(device="cuda").manual_seed(2), 50_000, 96, 4, "bf16", torch.int32)
    first = [t.clone() for t in _run(accelerator, logits, chosen)]
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, _run(accelerator, logits, chosen)))


def test_refusals(accelerator):
    logits, chosen = torch.zeros(6, 8, device="cuda"), torch.zeros(6, 2, dtype=torch.int64, device="cuda")
    loss, counts, p = torch.full((1,), 5.0, device="cuda"), torch.zeros(9, dtype=torch.int32, device="cuda"), torch.zeros(8, device="cuda")
    temp = accelerator.Allocate1D(accelerator.ComputeBalanceLossTempStorageSize(8, 6), torch.int32)
    good = dict(logits=logits, experts=chosen, mask=None, loss=loss, counts=counts, probabilities=p, temp=temp)
    balance, gradient = accelerator.CreateBalanceLoss(1.0), accelerator.CreateBalanceLossGradient(1.0, 2)
    mask = torch.ones(6, dtype=torch.bool, device="cuda")
    for changed, error in [
        (dict(logits=None), ib.ArgumentNullException), (dict(logits=logits.double()), ib.NotSupportedException), (dict(logits=logits[0]), ib.ArgumentOutOfRangeException),
        (dict(experts=chosen.float()), ib.NotSupportedException), (dict(experts=chosen[:5]), ib.ArgumentOutOfRangeException), (dict(mask=mask[:5]), ib.ArgumentOutOfRangeException),
        (dict(mask=mask.float()), ib.InvalidOperationException), (dict(counts=counts[:8]), ib.ArgumentOutOfRangeException), (dict(counts=counts.long()), ib.InvalidOperationException),
        (dict(probabilities=p[:7]), ib.ArgumentOutOfRangeException), (dict(loss=loss[:0]), ib.ArgumentOutOfRangeException), (dict(temp=temp[:-1]), ib.ArgumentOutOfRangeException),
        (dict(experts=chosen.cpu()), ib.InvalidOperationException), (dict(experts=chosen[:, :0]), ib.B200AlgException),
        (dict(logits=torch.zeros(6, 1_025, device="cuda"), counts=counts.new_zeros(1_026), probabilities=p.new_zeros(1_025)), ib.NotSupportedException),
    ]:
        with pytest.raises(error):
            balance(None, *(good | changed).values())
    good = dict(logits=logits, mask=None, counts=counts, lossGradient=loss, logitsGradient=torch.zeros_like(logits))
    for changed, error in [
        (dict(logitsGradient=None), ib.ArgumentNullException), (dict(logitsGradient=logits.half()), ib.InvalidOperationException), (dict(logitsGradient=logits[:5]), ib.ArgumentOutOfRangeException),
        (dict(lossGradient=loss.double()), ib.InvalidOperationException), (dict(counts=counts[:8]), ib.ArgumentOutOfRangeException), (dict(mask=mask.long()), ib.InvalidOperationException),
    ]:
        with pytest.raises(error):
            gradient(None, *(good | changed).values())
    assert float(loss) == 5.0
