"""Calls at the edges of what the operators of a training step document: temps of other sizes, empty calls, values at the ends of
their ranges."""
import pytest
import torch

import ilgpu_b200 as ib
from ilgpu_b200 import _native as N

from .training import TYPES, assert_within, clipped, embedding_gradient

pytestmark = pytest.mark.gpu


def test_a_temp_for_the_longest_batch_serves_the_shorter_ones(accelerator):
    gen = torch.Generator(device="cuda").manual_seed(11)
    rows, width, most = 900, 512, 33_000
    upstream = torch.randn(most, width, generator=gen, device="cuda").to(torch.bfloat16)
    temp = accelerator.Allocate1D(accelerator.ComputeEmbeddingGradientTempStorageSize(rows, width, most), torch.int32)
    call = accelerator.CreateEmbeddingGradient()
    for n in (33_000, 28_288, 28_289, 16_384, 14_144, 8_192, 7_073, 7_000, 1_025, 600, 1, 0):
        tokens = (torch.rand(n, generator=gen, device="cuda") ** 3 * rows).long()
        for narrow in (width, 40):
            temp.fill_(-1)
            out = torch.full((rows, narrow), float("nan"), device="cuda")
            call(None, tokens, upstream[:, :narrow], out, temp)
            accelerator.CheckDeviceStatus(None, temp)
            assert_within(out, *embedding_gradient(tokens, upstream[:, :narrow], 1.0, rows, torch.float32))


@pytest.mark.parametrize("types", ["bf16 fp32", "fp32 fp32", "bf16 bf16"])
@pytest.mark.parametrize("n, width", [(1_025, 1), (3_000, 33), (7_104, 2_051), (14_208, 512), (60_000, 9), (120_000, 64)])
def test_nothing_is_written_behind_the_temp(accelerator, n, width, types):
    """Every row crosses tiles, so that all shares are written."""
    source, target = (TYPES[t] for t in types.split())
    gen = torch.Generator(device="cuda").manual_seed(n)
    ints = accelerator.ComputeEmbeddingGradientTempStorageSize(3, width, n)
    whole = torch.full((ints + 4_096,), 0x5A5A5A5A, dtype=torch.int32, device="cuda")
    tokens = torch.randint(0, 3, (n,), generator=gen, device="cuda")
    upstream, out = torch.randn(n, width, generator=gen, device="cuda").to(source), torch.empty(3, width, dtype=target, device="cuda")
    accelerator.CreateEmbeddingGradient()(None, tokens, upstream, out, whole[:ints])
    assert_within(out, *embedding_gradient(tokens, upstream, 1.0, 3, target))
    assert bool((whole[ints:] == 0x5A5A5A5A).all())


@pytest.mark.parametrize("n, rows, width, accumulate", [(0, 5, 8, True), (0, 5, 8, False), (4, 0, 8, False), (4, 0, 8, True), (4, 5, 0, False), (0, 0, 0, True)])
def test_an_empty_gradient_leaves_a_status(accelerator, n, rows, width, accumulate):
    temp = torch.full((max(64, accelerator.ComputeEmbeddingGradientTempStorageSize(rows, width, n)),), -1, dtype=torch.int32, device="cuda")
    tokens, upstream = torch.zeros(n, dtype=torch.int64, device="cuda"), torch.ones(n, width, device="cuda")
    accelerator.CreateEmbeddingGradient(accumulate)(None, tokens, upstream, torch.empty(rows, width, device="cuda"), temp)
    accelerator.CheckDeviceStatus(None, temp)


@pytest.mark.parametrize("lengths", [[], [0, 0], [1], [5, 70_000], [3] * 100, [3] * 1_500])
def test_norm_and_clipping_leave_a_status(accelerator, lengths):
    views, out = [torch.ones(n, device="cuda") for n in lengths], torch.empty(1, device="cuda")
    temp = torch.empty(accelerator.ComputeGradientNormTempStorageSize(len(views)), dtype=torch.int32, device="cuda")
    for call in (lambda: accelerator.CreateGradientNorm()(None, views, out, temp), lambda: accelerator.CreateGradientClip()(None, views, None, 1.0, out, temp)):
        temp.fill_(-1)
        call()
        accelerator.CheckDeviceStatus(None, temp)


@pytest.mark.parametrize("tokens, experts", [(0, 8), (5, 8), (1_000, 8), (3_000, 40), (20_000, 8)])
def test_the_balance_loss_leaves_a_status(accelerator, tokens, experts):
    temp = torch.full((accelerator.ComputeBalanceLossTempStorageSize(experts, tokens),), -1, dtype=torch.int32, device="cuda")
    loss, counts, p = torch.empty(1, device="cuda"), torch.empty(experts + 1, dtype=torch.int32, device="cuda"), torch.empty(experts, device="cuda")
    accelerator.CreateBalanceLoss(1.0)(None, torch.zeros(tokens, experts, device="cuda"), torch.zeros(tokens, 2, dtype=torch.int64, device="cuda"), None, loss, counts, p, temp)
    accelerator.CheckDeviceStatus(None, temp)


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("choices", [(1 << 32) + 2, (1 << 31) + 2, (1 << 64) + 2, 1_025, 0, -1, 2 - (1 << 32)])
def test_choices_are_not_cut_to_a_word(monkeypatch, native, choices):
    if not native:
        monkeypatch.setattr(N, "_host", N._NoHostPath())
    accelerator = ib.Accelerator(0)
    logits, counts = torch.zeros(6, 8, device="cuda"), torch.tensor([3, 1, 1, 1, 2, 2, 1, 1, 6], dtype=torch.int32, device="cuda")
    gradient = torch.full_like(logits, 7.0)
    with pytest.raises((ib.ArgumentOutOfRangeException, ib.NotSupportedException, ib.B200AlgException)):
        accelerator.CreateBalanceLossGradient(1.0, choices)(None, logits, None, counts, torch.ones(1, device="cuda"), gradient)
    assert bool((gradient == 7.0).all())


@pytest.mark.parametrize("types", ["bf16 bf16", "fp32 fp32", "fp32 fp16"])
@pytest.mark.parametrize("scale", [float("inf"), float("nan"), -2.0, 1e300])
@pytest.mark.parametrize("width", [64, 33])
def test_a_token_without_a_row_gets_zeros_whatever_the_scale(accelerator, width, scale, types):
    source, target = (TYPES[t] for t in types.split())
    out = torch.full((3, width), 7.0, dtype=target, device="cuda")
    accelerator.CreateEmbedding()(None, torch.ones(4, width, dtype=source, device="cuda"), torch.tensor([-1, 2, 4], device="cuda"), out, scale)
    assert not bool(out[[0, 2]].any()) and not bool(torch.signbit(out[[0, 2]]).any())
    assert torch.equal(out[1].nan_to_num(7.0), torch.full((width,), scale, dtype=torch.float64, device="cuda").float().to(target).nan_to_num(7.0))


@pytest.mark.parametrize("types", ["fp32 fp32", "fp32 bf16", "bf16 fp32", "bf16 bf16"])
@pytest.mark.parametrize("given, max_norm", [(3e38, 1.0), (3e38, 3e-3), (3e38, 1e-7), (1e38, 1e-20), (1e20, 1e-19), (1e30, 1e-37), (3e38, 0.0), (1e-30, 1e-44), (2e37, 0.2)])
def test_factors_below_the_normal_numbers(accelerator, given, max_norm, types):
    """max_norm / norm may be a number that float holds with few bits, or not at all, while the products are ordinary numbers."""
    source, target = (TYPES[t] for t in types.split())
    gen = torch.Generator(device="cuda").manual_seed(13)
    sizes = torch.rand(5_001, generator=gen, device="cuda").mul_(80.0).sub_(80.0).exp_()  # all the way down to subnormal products
    view = (torch.randn(5_001, generator=gen, device="cuda").clamp_(-1.0, 1.0) * given * sizes).to(source)
    before, norm = view.clone(), torch.tensor([given], device="cuda")
    out = torch.empty_like(view, dtype=target)
    accelerator.CreateGradientScale()(None, [view], [out], max_norm, norm)
    assert_within(out, *clipped(before, float(norm), max_norm, target))
    if source == target:
        accelerator.CreateGradientScale()(None, [view], None, max_norm, norm)
        assert torch.equal(view, out)


def test_clipping_of_the_largest_gradients(accelerator):
    view, norm = torch.tensor([1e38, -2e38, 3e37, 1.0, 0.0], device="cuda"), torch.empty(1, device="cuda")
    before, temp = view.clone(), torch.empty(accelerator.ComputeGradientNormTempStorageSize(1), dtype=torch.int32, device="cuda")
    accelerator.CreateGradientClip()(None, [view], None, 1.0, norm, temp)
    assert_within(view, *clipped(before, float(norm), 1.0, torch.float32))
