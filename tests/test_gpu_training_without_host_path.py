"""The operators of a training step without the native host path (_host.so): algorithms.py alone gives the same bits."""
import pytest
import torch

import ilgpu_b200 as ib
from ilgpu_b200 import _native as N

from .training import TYPES, Balance, assert_within, clipped, embedding, embedding_gradient, norm

pytestmark = pytest.mark.gpu


class Fast:
    """The native path, and whether it has done the work."""

    def __init__(self, host):
        self.host, self.taken = host, []

    def __getattr__(self, name):
        def call(*arguments):
            done = getattr(self.host, name)(*arguments)
            self.taken.append(done)
            return done
        return call


@pytest.fixture
def both(monkeypatch):
    """An accelerator with the native path, which has to take every call, and one without."""
    host = Fast(ib.Accelerator(0)._host)
    monkeypatch.setattr(N, "_host", host)
    native = ib.Accelerator(0)
    monkeypatch.setattr(N, "_host", N._NoHostPath())
    yield native, ib.Accelerator(0)
    assert host.taken and all(host.taken)


def _matrix(gen, rows, width, dtype, stride):
    """Rows that are further apart than they are wide."""
    view = torch.zeros(rows, stride, dtype=dtype, device="cuda")[:, :width]
    view.copy_(torch.randn(rows, width, generator=gen, device="cuda"))
    return view


def _same(a, b):
    assert all(torch.equal(x, y) for x, y in zip(a, b, strict=True))


@pytest.mark.parametrize("stream", [False, True])
@pytest.mark.parametrize("source, target, ids", [("bf16", "fp32", torch.int32), ("fp32", "fp16", torch.int64)])
def test_embedding(both, source, target, ids, stream):
    gen = torch.Generator(device="cuda").manual_seed(1)
    rows, width, n = 90, 40, 700
    table, tokens = _matrix(gen, rows, width, TYPES[source], 44), torch.randint(-2, rows + 2, (2 * n,), generator=gen, device="cuda").to(ids)[::2]
    upstream, side = _matrix(gen, n + 3, width, TYPES[source], 56), torch.cuda.Stream() if stream else None
    torch.cuda.synchronize()
    results = []
    for acc in both:
        out, gradient = torch.zeros(n + 1, 48, dtype=TYPES[target], device="cuda")[:, :width], torch.full((rows, 41), 2.0, dtype=TYPES[target], device="cuda")[:, :width]
        temp = acc.Allocate1D(acc.ComputeEmbeddingGradientTempStorageSize(rows, width, n), torch.int32)
        added = gradient.clone()
        torch.cuda.synchronize()
        acc.CreateEmbedding()(side, table, tokens, out, 1.5)
        acc.CreateEmbeddingGradient()(side, tokens, upstream, gradient, temp, 0.75)
        acc.CreateEmbeddingGradient(accumulate=True)(side, tokens, upstream, added, temp, 0.75)
        acc.CheckDeviceStatus(side, temp)
        results.append((out, gradient, added))
    _same(*results)
    assert_within(results[0][0][:n], *embedding(table, tokens, 1.5, TYPES[target]))
    assert_within(results[0][1], *embedding_gradient(tokens, upstream, 0.75, rows, TYPES[target]))
    assert_within(results[0][2], *embedding_gradient(tokens, upstream, 0.75, rows, TYPES[target], torch.full((rows, width), 2.0)))


def test_norm_and_clipping(both):
    gen = torch.Generator(device="cuda").manual_seed(2)
    views = [torch.randn(s, generator=gen, device="cuda").to(TYPES[t]) for s, t in (((30, 7), "fp32"), ((5_000,), "bf16"), ((0,), "fp32"), ((3, 4, 5), "fp16"))]
    whole, results = norm(views), []
    for acc in both:
        temp = acc.Allocate1D(acc.ComputeGradientNormTempStorageSize(len(views)), torch.int32)
        outputs = [torch.empty_like(v, dtype=TYPES[t]) for v, t in zip(views, ("bf16", "fp32", "fp32", "fp32"))]
        again, place = [torch.empty_like(v) for v in views], [v.clone() for v in views]
        norms, given = torch.zeros(3, device="cuda"), torch.tensor([4.0 * whole], device="cuda")
        acc.CreateGradientNorm()(None, views, norms[:1], temp)
        acc.CreateGradientClip()(None, views, outputs, whole / 3, norms[1:2], temp)
        acc.CreateGradientClip()(None, place, None, whole / 5, norms[2:], temp)
        acc.CreateGradientScale()(None, tuple(views), tuple(again), whole, given)
        results.append([norms, *outputs, *place, *again])
    _same(*results)
    norms, outputs, place, again = results[0][0], results[0][1:5], results[0][5:9], results[0][9:]
    assert len(set(norms.tolist())) == 1
    for i, view in enumerate(views):
        assert_within(outputs[i], *clipped(view, float(norms[0]), whole / 3, outputs[i].dtype))
        assert_within(place[i], *clipped(view, float(norms[0]), whole / 5, view.dtype))
        assert_within(again[i], *clipped(view, float(given), whole, view.dtype))


@pytest.mark.parametrize("ids, masked", [(torch.int32, True), (torch.int64, False)])
def test_balance_loss(both, ids, masked):
    gen = torch.Generator(device="cuda").manual_seed(3)
    tokens, experts, choices = 300, 24, 3
    logits = _matrix(gen, tokens, experts, torch.bfloat16, 32)
    chosen = torch.zeros(tokens, 8, dtype=ids, device="cuda")[:, :choices]
    chosen.copy_(torch.randint(0, experts, (tokens, choices), generator=gen, device="cuda"))
    mask = torch.rand(tokens, generator=gen, device="cuda") < 0.7 if masked else None
    results = []
    for acc in both:
        loss, counts, p = torch.empty(1, device="cuda"), torch.empty(experts + 1, dtype=torch.int32, device="cuda"), torch.empty(experts, device="cuda")
        temp = acc.Allocate1D(acc.ComputeBalanceLossTempStorageSize(experts, tokens), torch.int32)
        acc.CreateBalanceLoss(0.02)(None, logits, chosen, mask, loss, counts, p, temp)
        gradient, added, upstream = torch.empty_like(logits), torch.ones(tokens, 40, dtype=torch.bfloat16, device="cuda")[:, :experts], torch.full((1,), 500.0, device="cuda")
        acc.CreateBalanceLossGradient(0.02, choices)(None, logits, mask, counts, upstream, gradient)
        acc.CreateBalanceLossGradient(0.02, choices, accumulate=True)(None, logits, mask, counts, upstream, added)
        results.append((loss, counts, p, gradient, added))
    _same(*results)
    loss, counts, p, gradient, added = results[0]
    b = Balance(logits, chosen, mask, 0.02)
    value, bound, mean, off = b.loss()
    assert_within(loss, value, bound)
    assert_within(p, mean, off)
    assert counts.tolist() == b.counts.tolist() + [b.number]
    assert_within(gradient, *b.gradient(500.0, torch.bfloat16))
    assert_within(added, *b.gradient(500.0, torch.bfloat16, base=torch.ones(tokens, experts)))
