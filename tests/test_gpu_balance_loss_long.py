"""The balance loss of so many tokens that a lane's sums in 32 bits go on in 64 several times.

The rows repeat a pattern, so that the definition in 64 bits takes each of its rows as often as it comes.  The bounds are
those of tests/training.py: 128 additions in 32 bits and then 64, however many tokens there are."""
import pytest
import torch

from .training import TYPES, U, Balance, assert_within

pytestmark = pytest.mark.gpu
COEFFICIENT = 0.01


def _check(acc, tokens, pattern, chosen, mask=None):
    """`pattern`, `chosen` and `mask` repeated up to `tokens` rows."""
    size, experts = pattern.shape
    times = torch.full((size,), tokens // size, dtype=torch.float64)
    times[:tokens % size] += 1
    repeat = lambda t: t.repeat(-(-tokens // size), *[1] * (t.dim() - 1))[:tokens]  # noqa: E731
    loss, counts, p = torch.empty(1, device="cuda"), torch.empty(experts + 1, dtype=torch.int32, device="cuda"), torch.empty(experts, device="cuda")
    temp = acc.Allocate1D(acc.ComputeBalanceLossTempStorageSize(experts, tokens), torch.int32)
    temp.fill_(-1)
    acc.CreateBalanceLoss(COEFFICIENT)(None, repeat(pattern), repeat(chosen), None if mask is None else repeat(mask), loss, counts, p, temp)
    b = Balance(pattern, chosen, mask, COEFFICIENT)
    times = times * b.valid
    number = int(times.sum())
    weights = torch.zeros(experts, dtype=torch.float64)
    weights.index_add_(0, chosen.cpu().long().flatten(), times.repeat_interleave(chosen.shape[1]))
    assert counts.tolist() == weights.long().tolist() + [number]
    mean = (b.p * times[:, None]).sum(dim=0) / number
    off = (b.p * b.relative * times[:, None]).sum(dim=0) / number + 130 * U * mean + 2.0 ** -120
    assert_within(p, mean, off + U * mean)
    share = COEFFICIENT * experts * weights / number / chosen.shape[1]
    value, bound = (share * mean).sum().reshape(1), (share * off).sum().reshape(1)
    assert_within(loss, value, bound + 2 * U * value)


@pytest.mark.parametrize("seed", [2, 3])
def test_the_error_does_not_grow_with_the_tokens(accelerator, seed):
    """One row over and over: each addition in 32 bits is off to the same side as long as the sum has the same exponent, which
    adds up to hundreds of U over the 1770 rows that a lane sees."""
    row = torch.randn(1, 8, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).cuda()
    _check(accelerator, (1 << 27) + 12_345, row, torch.tensor([[3]], dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("kind, tokens, experts, choices", [
    ("fp32", 40_000_003, 8, 2), ("bf16", 10_000_007, 64, 2), ("fp16", 3_000_000, 60, 3), ("bf16", 700_001, 1_024, 4), ("fp32", 1_200_000, 300, 2),
    ("bf16", 2_500_000, 99, 2), ("fp32", 600_011, 1_021, 1)])
def test_many_stretches(accelerator, kind, tokens, experts, choices):
    gen = torch.Generator(device="cuda").manual_seed(experts)
    size = 1_009
    pattern = (torch.randn(size, experts, generator=gen, device="cuda") * 2.0).to(TYPES[kind])
    chosen = torch.randint(0, experts, (size, choices), generator=gen, device="cuda").to(torch.int32)
    mask = torch.rand(size, generator=gen, device="cuda") < 0.8
    _check(accelerator, tokens, pattern, chosen)
    pattern[~mask] = float("nan")
    _check(accelerator, tokens, pattern, chosen, mask)
