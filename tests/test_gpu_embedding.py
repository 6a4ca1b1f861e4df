"""The embedding lookup and its gradient by sorted tokens, against their definitions in 64 bits."""
import pytest
import torch

import ilgpu_b200 as ib

from .training import TYPES, assert_within, embedding, embedding_gradient

pytestmark = pytest.mark.gpu


def _matrix(gen, rows, width, dtype, stride=None, offset=0, size=1.0):
    """A matrix whose rows are `stride` apart and whose first element lies `offset` elements behind a boundary; between the rows lie NaNs."""
    stride = width if stride is None else stride
    flat = torch.full((offset + max(rows, 1) * stride,), float("nan"), dtype=dtype, device="cuda")
    view = flat[offset:].as_strided((rows, width), (stride, 1))
    view.copy_(torch.randn(rows, width, generator=gen, device="cuda") * size)
    return flat, view


def _tokens(gen, n, rows, kind, dtype, stride=1):
    if kind == "uniform":
        t = torch.randint(0, max(rows, 1), (n,), generator=gen, device="cuda")
    elif kind == "few":       # long runs
        t = torch.randint(0, min(3, rows), (n,), generator=gen, device="cuda")
    elif kind == "one":
        t = torch.full((n,), rows - 1, device="cuda")
    elif kind == "outside":   # some without a row, on both sides
        t = torch.randint(-rows, 2 * rows, (n,), generator=gen, device="cuda")
    elif kind == "none":
        t = torch.full((n,), -1, device="cuda")
    else:                     # the ends of the range, and values whose low 32 bits are in it
        info = torch.iinfo(dtype)
        values = [info.min, info.max, -1, 0, rows - 1, rows] + ([1 << 32, (1 << 32) + 1, -(1 << 32)] if dtype == torch.int64 else [])
        t = torch.tensor(values, device="cuda")[torch.randint(0, len(values), (n,), generator=gen, device="cuda")]
    out = torch.zeros(max(n, 1) * stride, dtype=dtype, device="cuda")[::stride][:n]
    out.copy_(t.to(dtype))
    return out


def _same_gaps(flat, view, stride, offset, before):
    """Nothing but the rows has changed."""
    rows, width = view.shape
    inside = torch.zeros_like(flat, dtype=torch.bool)
    inside[offset:].as_strided((rows, width), (stride, 1)).fill_(True)
    bits = torch.int16 if flat.element_size() == 2 else torch.int32
    assert torch.equal(flat.view(bits)[~inside], before.view(bits)[~inside])


SHAPES = [  # tokens, rows, width
    (1, 1, 1), (1, 5, 8), (3, 7, 33), (8, 100, 4096), (65, 1000, 64), (257, 50, 1000), (1000, 3, 7), (513, 2048, 1024), (40, 17, 12), (5, 9, 20_001),
]


@pytest.mark.parametrize("types", ["bf16 bf16", "fp32 bf16", "bf16 fp32", "fp16 fp16", "fp32 fp32", "fp16 bf16", "fp32 fp16"])
@pytest.mark.parametrize("n, rows, width", SHAPES)
def test_lookup(accelerator, types, n, rows, width):
    source, target = (TYPES[t] for t in types.split())
    gen = torch.Generator(device="cuda").manual_seed(n * 7 + width)
    _, table = _matrix(gen, rows, width, source)
    for kind, dtype, scale in (("uniform", torch.int32, 1.0), ("outside", torch.int64, 5.7), ("extreme", torch.int64, -0.125), ("extreme", torch.int32, 1.0)):
        tokens = _tokens(gen, n, rows, kind, dtype)
        out = torch.full((n, width), float("nan"), dtype=target, device="cuda")
        accelerator.CreateEmbedding()(None, table, tokens, out, scale)
        assert_within(out, *embedding(table, tokens, scale, target))


@pytest.mark.parametrize("width, stride, offset, out_stride, out_offset", [
    (64, 64, 1, 64, 0), (64, 72, 0, 80, 0), (64, 65, 0, 67, 3), (64, 68, 4, 64, 0), (63, 64, 0, 64, 0), (1, 5, 2, 3, 1), (8, 8, 8, 24, 16)])
@pytest.mark.parametrize("types", ["bf16 bf16", "fp32 fp16", "fp32 fp32"])
def test_lookup_in_strided_views(accelerator, types, width, stride, offset, out_stride, out_offset):
    source, target = (TYPES[t] for t in types.split())
    gen = torch.Generator(device="cuda").manual_seed(width + stride)
    n, rows = 77, 50
    _, table = _matrix(gen, rows, width, source, stride, offset)
    flat, out = _matrix(gen, n + 3, width, target, out_stride, out_offset)
    tokens = _tokens(gen, n, rows, "outside", torch.int64, stride=3)
    before, behind = flat.clone(), out[n:].clone()
    accelerator.CreateEmbedding()(None, table, tokens, out, 2.0)
    assert_within(out[:n], *embedding(table, tokens, 2.0, target))
    assert torch.equal(out[n:], behind)  # rows behind the last token stay
    _same_gaps(flat, out, out_stride, out_offset, before)


def test_lookup_passes_on_what_is_not_finite(accelerator):
    table = torch.tensor([[1.0, float("inf"), -float("inf"), float("nan")], [1e38, -1e38, 1e-45, 0.0]], device="cuda")
    out = torch.empty(2, 4, dtype=torch.float16, device="cuda")
    accelerator.CreateEmbedding()(None, table, torch.tensor([0, 1], device="cuda"), out, 1.0)
    assert torch.equal(out.nan_to_num(nan=7.0), table.to(torch.float16).nan_to_num(nan=7.0))


def test_lookup_of_nothing(accelerator):
    out = torch.full((4, 8), 3.0, device="cuda")
    accelerator.CreateEmbedding()(None, torch.ones(5, 8, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda"), out)
    assert bool((out == 3.0).all())
    accelerator.CreateEmbedding()(None, torch.empty(0, 8, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"), out)  # no row at all
    assert bool((out[:2] == 0.0).all()) and bool((out[2:] == 3.0).all())


def test_lookup_past_32_bits_of_elements(accelerator):
    """Rows that begin behind 2^32 elements of the table and of the output."""
    rows, width, n = 70_000, 65_536, 66_000
    table = torch.zeros(rows, width, dtype=torch.bfloat16, device="cuda")
    marks = torch.arange(rows, device="cuda")
    table[:, 0] = (marks % 251).to(torch.bfloat16)
    table[:, -1] = (marks % 241).to(torch.bfloat16)
    tokens = (torch.arange(n, device="cuda") * 7 + 69_000) % rows
    out = torch.empty(n, width, dtype=torch.bfloat16, device="cuda")
    accelerator.CreateEmbedding()(None, table, tokens, out)
    assert torch.equal(out[:, 0], (tokens % 251).to(torch.bfloat16)) and torch.equal(out[:, -1], (tokens % 241).to(torch.bfloat16))
    assert not bool(out[:, 1:-1].any())


def test_lookup_of_more_groups_than_one_launch_counts(accelerator):
    n = (1 << 30) + 5_000
    table = torch.tensor([[1.0, -1.0], [2.0, -2.0], [3.0, -3.0]], dtype=torch.bfloat16, device="cuda")
    tokens = torch.arange(n, dtype=torch.int32, device="cuda").remainder_(5).sub_(1)
    out = torch.full((n, 2), 7.0, dtype=torch.bfloat16, device="cuda")
    accelerator.CreateEmbedding()(None, table, tokens, out)
    want = torch.where(tokens > 2, 0, tokens + 1).to(torch.bfloat16)
    assert torch.equal(out[:, 0], want) and torch.equal(out[:, 1], -want)


def _gradient(acc, tokens, upstream, out, scale=1.0, accumulate=False, stream=None):
    temp = acc.Allocate1D(acc.ComputeEmbeddingGradientTempStorageSize(out.shape[0], out.shape[1], tokens.numel()), torch.int32)
    temp.fill_(-1)  # whatever was there
    acc.CreateEmbeddingGradient(accumulate)(stream, tokens, upstream, out, temp, scale)
    if tokens.numel() and out.numel():
        acc.CheckDeviceStatus(stream, temp)


GRADIENT_SHAPES = [  # tokens, rows, width: one token, tiles of every length, runs over several tiles, wide and narrow rows
    (1, 1, 1), (1, 40, 8), (2, 3, 5), (15, 4, 64), (16, 100, 64), (17, 3, 33), (129, 9, 48), (300, 2000, 768), (2_367, 31, 40), (2_368, 5, 8),
    (4_737, 700, 129), (20_000, 37, 24), (19_001, 5000, 64), (500, 300, 4_100), (512, 90, 72), (513, 90, 72), (5_000, 30_000, 256), (60_000, 9, 16),
    (3_000, 50_000, 33), (10_000, 77, 2_051), (2_000_003, 5_000, 8),
    (1_024, 300, 64), (1_025, 300, 64), (900, 40, 261), (90, 700, 9_001),
]


@pytest.mark.parametrize("types", ["bf16 fp32", "bf16 bf16", "fp32 fp32", "fp16 fp32", "fp16 fp16", "fp32 bf16"])
@pytest.mark.parametrize("n, rows, width", GRADIENT_SHAPES)
def test_gradient(accelerator, types, n, rows, width):
    source, target = (TYPES[t] for t in types.split())
    gen = torch.Generator(device="cuda").manual_seed(n + rows + width)
    _, upstream = _matrix(gen, n, width, source)
    for kind, dtype, scale in (("uniform", torch.int32, 1.0), ("few", torch.int64, 0.3), ("outside", torch.int64, -2.0), ("one", torch.int32, 1.0),
                               ("none", torch.int32, 1.0), ("extreme", torch.int64, 1.0)):
        tokens = _tokens(gen, n, rows, kind, dtype)
        out = torch.full((rows, width), float("nan"), dtype=target, device="cuda")
        _gradient(accelerator, tokens, upstream, out, scale)
        exact, bound = embedding_gradient(tokens, upstream, scale, rows, target)
        if target != torch.float16 or float(exact.abs().max()) < 65_000:
            assert_within(out, exact, bound)


@pytest.mark.parametrize("types", ["bf16 fp32", "fp32 fp16", "bf16 bf16"])
@pytest.mark.parametrize("n, rows, width, kind", [(1, 5, 8, "uniform"), (700, 900, 72, "uniform"), (5_000, 60, 31, "outside"), (3_000, 10, 256, "few"), (64, 10, 8, "none")])
def test_gradient_added_to_what_is_there(accelerator, types, n, rows, width, kind):
    source, target = (TYPES[t] for t in types.split())
    gen = torch.Generator(device="cuda").manual_seed(n)
    _, upstream = _matrix(gen, n, width, source)
    tokens = _tokens(gen, n, rows, kind, torch.int32)
    out = torch.randn(rows, width, generator=gen, device="cuda").to(target)
    before = out.clone()
    _gradient(accelerator, tokens, upstream, out, 0.5, accumulate=True)
    assert_within(out, *embedding_gradient(tokens, upstream, 0.5, rows, target, before))
    named = torch.zeros(rows, dtype=torch.bool, device="cuda")
    named[tokens[(tokens >= 0) & (tokens < rows)].long()] = True
    assert torch.equal(out[~named], before[~named])


@pytest.mark.parametrize("width, stride, offset, out_stride, out_offset", [(64, 64, 1, 64, 0), (64, 72, 8, 80, 0), (64, 65, 0, 67, 3), (63, 64, 0, 64, 0), (1, 5, 2, 3, 1)])
@pytest.mark.parametrize("types", ["bf16 fp32", "fp32 bf16"])
def test_gradient_in_strided_views(accelerator, types, width, stride, offset, out_stride, out_offset):
    source, target = (TYPES[t] for t in types.split())
    gen = torch.Generator(device="cuda").manual_seed(width + stride)
    rows = 150
    for n in (300, 700):  # with and without a sort
        _, upstream = _matrix(gen, n + 2, width, source, stride, offset)
        flat, out = _matrix(gen, rows, width, target, out_stride, out_offset)
        tokens = _tokens(gen, n, rows, "outside", torch.int32, stride=2)
        before = flat.clone()
        _gradient(accelerator, tokens, upstream, out, 3.0)
        assert_within(out, *embedding_gradient(tokens, upstream, 3.0, rows, target))
        _same_gaps(flat, out, out_stride, out_offset, before)


@pytest.mark.parametrize("n", [300, 3_000])
def test_upstream_rows_without_a_row_of_the_table_are_not_read(accelerator, n):
    upstream = torch.full((n, 24), float("nan"), device="cuda")
    tokens = torch.full((n,), -1, dtype=torch.int64, device="cuda")
    upstream[7], tokens[7] = 2.0, 4
    out = torch.empty(6, 24, device="cuda")
    _gradient(accelerator, tokens, upstream, out)
    assert bool((out[4] == 2.0).all()) and not bool(out[[0, 1, 2, 3, 5]].any())


def test_gradient_of_nothing(accelerator):
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    out = torch.full((5, 8), 3.0, device="cuda")
    _gradient(accelerator, none, torch.empty(0, 8, device="cuda"), out, accumulate=True)
    assert bool((out == 3.0).all())
    _gradient(accelerator, none, torch.empty(0, 8, device="cuda"), out)
    assert not bool(out.any())
    _gradient(accelerator, torch.zeros(4, dtype=torch.int64, device="cuda"), torch.ones(4, 8, device="cuda"), torch.empty(0, 8, device="cuda"))


def test_gradient_bits_do_not_change(accelerator):
    gen = torch.Generator(device="cuda").manual_seed(5)
    n, rows, width = 30_000, 200, 264
    upstream = torch.randn(n, width, generator=gen, device="cuda").to(torch.bfloat16)
    tokens = (torch.rand(n, generator=gen, device="cuda") ** 4 * rows).long()
    first = torch.empty(rows, width, device="cuda")
    _gradient(accelerator, tokens, upstream, first)
    for _ in range(5):
        again = torch.empty_like(first)
        _gradient(accelerator, tokens, upstream, again)
        assert torch.equal(first, again)


@pytest.mark.parametrize("n", [400, 6_000])
def test_what_is_not_finite_stays_in_its_row_and_column(accelerator, n):
    gen = torch.Generator(device="cuda").manual_seed(3)
    upstream = torch.randn(n, 37, generator=gen, device="cuda")
    tokens = torch.randint(0, 50, (n,), generator=gen, device="cuda")
    upstream[7, 5], upstream[9, 36], upstream[11, 0] = float("nan"), float("inf"), -float("inf")
    out = torch.empty(50, 37, device="cuda")
    _gradient(accelerator, tokens, upstream, out)
    exact, bound = embedding_gradient(tokens, upstream, 1.0, 50, torch.float32)
    assert_within(out, exact, torch.where(bound.isfinite(), bound, 0.0))
    assert int((~out.isfinite()).sum()) == 3


@pytest.mark.parametrize("n", [300, 6_000, 60_000])
def test_calls_in_a_row_over_the_same_buffers(accelerator, n):
    """What clears rows starts while the sort runs: not before the kernel that reads the last call's result, or writes the
    tokens, is through."""
    gen = torch.Generator(device="cuda").manual_seed(n)
    rows, width = 20_000, 128
    sets = [(torch.randint(0, rows, (n,), generator=gen, device="cuda"), torch.randn(n, width, generator=gen, device="cuda")) for _ in range(3)]
    out, temp = torch.empty(rows, width, device="cuda"), accelerator.Allocate1D(accelerator.ComputeEmbeddingGradientTempStorageSize(rows, width, n), torch.int32)
    call, want = accelerator.CreateEmbeddingGradient(), []
    for tokens, upstream in sets:
        call(None, tokens, upstream, out, temp)
        torch.cuda.synchronize()
        want.append(out.clone())
        assert_within(out, *embedding_gradient(tokens, upstream, 1.0, rows, torch.float32))
    tokens, seen = torch.empty_like(sets[0][0]), []
    for i in range(12):
        tokens.copy_(sets[i % 3][0])
        call(None, tokens, sets[i % 3][1], out, temp)
        seen.append(out * 1.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for i in range(3):
            tokens.copy_(sets[i][0])
            call(None, tokens, sets[i][1], out, temp)
            seen[i].copy_(out)
    torch.cuda.synchronize()
    assert all(torch.equal(s, want[i % 3]) for i, s in enumerate(seen))
    for s in seen[:3]:
        s.zero_()
    for _ in range(4):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(s, w) for s, w in zip(seen, want))
    del graph


def test_gradient_is_the_lookups(accelerator):
    """Against differences: <lookup(table + d) - lookup(table), g> = <d, gradient(g)>, exactly linear."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    n, rows, width, scale = 3_000, 411, 96, 1.75
    tokens = _tokens(gen, n, rows, "outside", torch.int64)
    table, d = (torch.randint(-64, 65, (rows, width), generator=gen, device="cuda").float() for _ in range(2))  # whole numbers: no rounding
    g = torch.randint(-8, 9, (n, width), generator=gen, device="cuda").float()
    out, moved, gradient = torch.empty(n, width, device="cuda"), torch.empty(n, width, device="cuda"), torch.empty(rows, width, device="cuda")
    embed = accelerator.CreateEmbedding()
    embed(None, table, tokens, out, scale)
    embed(None, table + d, tokens, moved, scale)
    _gradient(accelerator, tokens, g, gradient, scale)
    assert float(((moved - out).double() * g.double()).sum()) == float((d.double() * gradient.double()).sum())


def test_refusals(accelerator):
    embed, gradient = accelerator.CreateEmbedding(), accelerator.CreateEmbeddingGradient()
    table, tokens, out = torch.ones(5, 8, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda"), torch.ones(3, 8, device="cuda")
    temp = accelerator.Allocate1D(accelerator.ComputeEmbeddingGradientTempStorageSize(5, 8, 3), torch.int32)
    for call, error in [
        (lambda: embed(None, None, tokens, out), ib.ArgumentNullException), (lambda: embed(None, table, tokens.float(), out), ib.NotSupportedException),
        (lambda: embed(None, table.double(), tokens, out), ib.NotSupportedException), (lambda: embed(None, table, tokens, out[:2]), ib.ArgumentOutOfRangeException),
        (lambda: embed(None, table, tokens, out[:, :7]), ib.ArgumentOutOfRangeException), (lambda: embed(None, table.cpu(), tokens, out), ib.InvalidOperationException),
        (lambda: embed(None, table.t(), tokens, out), ib.NotSupportedException), (lambda: embed(None, table[0], tokens, out), ib.ArgumentOutOfRangeException),
        (lambda: embed(None, table, tokens[None], out), ib.ArgumentOutOfRangeException), (lambda: embed(None, table, tokens, out[:1].expand(3, 8)), ib.ArgumentOutOfRangeException),
        (lambda: gradient(None, tokens, out[:2], table, temp), ib.ArgumentOutOfRangeException), (lambda: gradient(None, tokens, out, table, temp[:8]), ib.ArgumentOutOfRangeException),
        (lambda: gradient(None, tokens, out, table, None), ib.ArgumentNullException), (lambda: gradient(None, tokens, out, table, temp[1:]), (ib.InvalidOperationException, ib.ArgumentOutOfRangeException)),
        (lambda: gradient(None, tokens.short(), out, table, temp), ib.NotSupportedException), (lambda: gradient(None, tokens, out.long(), table, temp), ib.NotSupportedException),
    ]:
        with pytest.raises(error):
            call()
    assert bool((out == 1.0).all()) and bool((table == 1.0).all())
