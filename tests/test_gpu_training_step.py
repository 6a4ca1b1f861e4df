"""The operators of a training step together, as a program uses them: tokens are looked up, a router sees the rows and its
balance loss is taken, the gradients come back through the router to the table, all of them are clipped by their common
norm.  Run eagerly, on another stream, captured into a graph and replayed, and from two streams at once."""
import pytest
import torch

from .training import NORM_BOUND, U, Balance, assert_within, clipped, embedding, embedding_gradient, norm

pytestmark = pytest.mark.gpu
ROWS, WIDTH, TOKENS, EXPERTS, CHOICES, SCALE, COEFFICIENT, MAX_NORM = 500, 64, 1_200, 16, 2, 8.0, 0.02, 0.05


class Step:
    def __init__(self, acc, seed, tokens=TOKENS):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.acc, self.gen = acc, gen
        self.table = torch.randn(ROWS, WIDTH, generator=gen, device="cuda").mul_(0.1).to(torch.bfloat16)
        self.router = torch.randn(WIDTH, EXPERTS, generator=gen, device="cuda").mul_(0.2)
        self.tokens = torch.empty(tokens, dtype=torch.int64, device="cuda")
        self.rows, self.logits = torch.empty(tokens, WIDTH, device="cuda"), torch.empty(tokens, EXPERTS, device="cuda")
        self.chosen = torch.empty(tokens, CHOICES, dtype=torch.int64, device="cuda")
        self.loss, self.counts, self.mean = torch.empty(1, device="cuda"), torch.empty(EXPERTS + 1, dtype=torch.int32, device="cuda"), torch.empty(EXPERTS, device="cuda")
        self.one, self.d_logits, self.d_rows = torch.ones(1, device="cuda"), torch.empty(tokens, EXPERTS, device="cuda"), torch.empty(tokens, WIDTH, device="cuda")
        self.gradients = [torch.empty(ROWS, WIDTH, device="cuda"), torch.empty(WIDTH, EXPERTS, device="cuda")]
        self.clipped, self.norm = [torch.empty(ROWS, WIDTH, dtype=torch.bfloat16, device="cuda"), torch.empty(WIDTH, EXPERTS, device="cuda")], torch.empty(1, device="cuda")
        self.mask = torch.empty(tokens, dtype=torch.bool, device="cuda")
        temp = lambda ints: acc.Allocate1D(ints, torch.int32)  # noqa: E731
        self.temps = (temp(acc.ComputeBalanceLossTempStorageSize(EXPERTS, tokens)), temp(acc.ComputeEmbeddingGradientTempStorageSize(ROWS, WIDTH, tokens)),
                      temp(acc.ComputeGradientNormTempStorageSize(2)))
        self.new_tokens()

    def new_tokens(self):
        n = self.tokens.numel()
        self.tokens.copy_((torch.rand(n, generator=self.gen, device="cuda") ** 3 * ROWS).long())
        self.tokens[n - n // 10:] = -1  # padding
        self.mask.copy_(self.tokens >= 0)

    def run(self, stream=None):
        acc = self.acc
        with torch.cuda.stream(stream):
            acc.CreateEmbedding()(stream, self.table, self.tokens, self.rows, SCALE)
            torch.mm(self.rows, self.router, out=self.logits)
            torch.topk(self.logits, CHOICES, dim=1, out=(torch.empty_like(self.logits[:, :CHOICES]), self.chosen))
            acc.CreateBalanceLoss(COEFFICIENT)(stream, self.logits, self.chosen, self.mask, self.loss, self.counts, self.mean, self.temps[0])
            acc.CreateBalanceLossGradient(COEFFICIENT, CHOICES)(stream, self.logits, self.mask, self.counts, self.one, self.d_logits)
            torch.mm(self.d_logits, self.router.t(), out=self.d_rows)
            torch.mm(self.rows.t(), self.d_logits, out=self.gradients[1])
            acc.CreateEmbeddingGradient()(stream, self.tokens, self.d_rows, self.gradients[0], self.temps[1], SCALE)
            acc.CreateGradientClip()(stream, self.gradients, self.clipped, MAX_NORM, self.norm, self.temps[2])

    def results(self):
        return [self.rows, self.loss, self.counts, self.mean, self.d_logits, *self.gradients, self.norm, *self.clipped]

    def check(self):
        torch.cuda.synchronize()
        assert_within(self.rows, *embedding(self.table, self.tokens, SCALE, torch.float32))
        b = Balance(self.logits, self.chosen, self.mask, COEFFICIENT)
        value, bound, mean, off = b.loss()
        assert_within(self.loss, value, bound)
        assert_within(self.mean, mean, off)
        assert self.counts.tolist() == b.counts.tolist() + [b.number]
        assert_within(self.d_logits, *b.gradient(1.0, torch.float32))
        assert_within(self.gradients[0], *embedding_gradient(self.tokens, self.d_rows, SCALE, ROWS, torch.float32))
        whole = norm(self.gradients)
        assert abs(float(self.norm) - whole) <= NORM_BOUND * whole
        for g, c in zip(self.gradients, self.clipped):
            assert_within(c, *clipped(g, float(self.norm), MAX_NORM, c.dtype))


def test_step(accelerator):
    step = Step(accelerator, 1)
    for _ in range(3):
        step.run()
        step.check()
        step.new_tokens()


def test_its_gradient_is_autograds(accelerator):
    """The whole chain against torch's own derivative of the definition in 64 bits."""
    step = Step(accelerator, 2)
    step.run()
    torch.cuda.synchronize()
    table, router = step.table.double().requires_grad_(), step.router.double().requires_grad_()
    rows = torch.where(step.mask[:, None], table[step.tokens.clamp(min=0)] * SCALE, 0.0)
    p = torch.softmax(rows @ router, dim=1)[step.mask]
    loss = COEFFICIENT * EXPERTS * (step.counts[:EXPERTS].double() / (step.counts[EXPERTS] * CHOICES) * p.mean(dim=0)).sum()
    loss.backward()
    # products over 64 columns and 1200 rows and a softmax in 32 bits: some 10^-5 of the largest sums of magnitudes; a mistake in a factor is far over it
    assert float((step.loss.double() - loss.detach()).abs()) <= 1e-5 * float(loss.detach())
    for got, want in ((step.gradients[0], table.grad), (step.gradients[1], router.grad)):
        assert float((got.double() - want).norm()) <= 1e-3 * float(want.norm())


def test_on_another_stream(accelerator):
    step, want = Step(accelerator, 3), Step(accelerator, 3)
    want.run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    step.run(side)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    step.check()
    assert all(torch.equal(a, b) for a, b in zip(step.results(), want.results()))


@pytest.mark.parametrize("tokens", [TOKENS, 30_000])
def test_captured_and_replayed(accelerator, tokens):
    step, eager = Step(accelerator, 4, tokens), Step(accelerator, 4, tokens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    step.run(side)  # warm-up
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.run()
        step.run()  # twice over the same buffers
    for _ in range(3):
        for r in step.results():
            r.fill_(-1)
        graph.replay()
        eager.run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(step.results(), eager.results()))
        step.new_tokens()
        eager.new_tokens()
        torch.cuda.synchronize()
    del graph


def test_two_at_once(accelerator):
    """Calls whose workspaces are their own may overlap."""
    steps, streams = [Step(accelerator, s, 9_000) for s in (5, 6)], [torch.cuda.Stream() for _ in range(2)]
    for stream in streams:
        stream.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        for step, stream in zip(steps, streams):
            step.run(stream)
    torch.cuda.synchronize()
    for step in steps:
        step.check()
