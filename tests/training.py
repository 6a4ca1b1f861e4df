"""The operators of a training step from their definitions in 64 bits, on the CPU, with bounds on what the GPU's
arithmetic may be off by.  U is half a step of float; a type's own rounding is off by at most half of its eps, relative
to the value, and by half of its smallest number where that is more."""
import torch

U = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def rounding(dtype, value):
    """At most half a step of `dtype` at |value| (a little over, for the value itself is off by the bounds beside it)."""
    info = torch.finfo(dtype)
    return torch.clamp(1.01 * info.eps / 2 * value.abs(), min=info.smallest_normal * info.eps / 2)


def assert_within(got, exact, bound):
    got, exact, bound = got.detach().cpu().double(), exact.cpu().double(), bound.cpu().double()
    assert got.shape == exact.shape
    assert torch.equal(torch.isnan(got), torch.isnan(exact))
    off = (got - exact).abs()
    off[(got == exact) | torch.isnan(exact)] = 0.0
    worst = (off - bound).max() if off.numel() else torch.tensor(-1.0)
    assert worst <= 0.0, f"off by {off.flatten()[(off - bound).argmax()]:.3e}, at most {bound.expand_as(off).flatten()[(off - bound).argmax()]:.3e}"


def embedding(table, tokens, scale, dtype):
    """(values, bound): one product in float and one rounding."""
    table, tokens = table.cpu().double(), tokens.cpu().long()
    there = (tokens >= 0) & (tokens < table.shape[0])
    exact = torch.zeros(tokens.numel(), table.shape[1], dtype=torch.float64)
    exact[there] = table[tokens[there]] * scale
    return exact, 2 * U * exact.abs() + rounding(dtype, exact)  # the scale is rounded to float as well


def embedding_gradient(tokens, upstream, scale, rows, dtype, base=None):
    """(values, bound): m summands in any order are off by at most m U times the sum of their magnitudes."""
    upstream, tokens = upstream.cpu().double()[:tokens.numel()], tokens.cpu().long()
    there = ((tokens >= 0) & (tokens < rows)).nonzero().flatten()
    exact, size = (torch.zeros(rows, upstream.shape[1], dtype=torch.float64) for _ in range(2))
    exact.index_add_(0, tokens[there], upstream[there] * scale)
    size.index_add_(0, tokens[there], (upstream[there] * scale).abs())
    summands = torch.zeros(rows, dtype=torch.float64).index_add_(0, tokens[there], torch.ones(len(there), dtype=torch.float64))
    bound = (summands[:, None] + 3) * U * size
    if base is not None:
        exact = exact + base.cpu().double()
        bound = bound + U * (exact.abs() + size)
    return exact, bound + rounding(dtype, exact)


# The norm: each sum in 32 bits is over at most 64 squares, none negative: 65 U of it; they are joined in 64 bits, the root halves what
# is off, and the result is rounded to float.
NORM_BOUND = 34 * U


def norm(views):
    return sum(float(v.double().square().sum()) for v in views) ** 0.5


def clipped(view, norm, max_norm, dtype):
    """(values, bound) by the norm that the GPU found: the factor and the product are rounded to float."""
    factor = max_norm / norm if norm > max_norm else 1.0
    exact = view.cpu().double() * factor
    return exact, 2.01 * U * exact.abs() + 2.0 ** -149 + rounding(dtype, exact)


class Balance:
    """The balance loss and its gradient, and how far the GPU's may be off.

    x - max x is rounded (U), its product with log2 e as well, and log2 e itself (U each); 2^y is the GPU's approximation, off by 2^-22.
    So exp is off by 3 U |x - max x| + 4 U of itself; where that is not small, |x - max x| > 100, it is below 2^-126 and may be taken
    as zero.  The sum over a row of E is off by (E + 1) U more, its inverse and the product by 2 U."""

    def __init__(self, logits, chosen, mask, coefficient):
        x = logits.cpu().double()
        self.tokens, self.experts = x.shape
        self.choices, self.coefficient = chosen.shape[1], coefficient
        self.valid = torch.ones(self.tokens, dtype=torch.bool) if mask is None else mask.cpu().bool()[:self.tokens]
        x = torch.where(self.valid[:, None], x, 0.0)
        top = x.amax(dim=1, keepdim=True)
        top = torch.where(top == -torch.inf, 0.0, top)
        e = (x - top).exp()
        whole = e.sum(dim=1, keepdim=True)
        p = torch.where(whole == 0.0, 0.0, e / whole)
        self.p = torch.where(self.valid[:, None], p, 0.0)
        far = (top - x).clamp(0.0, 100.0).nan_to_num(0.0)
        mean_far = (torch.where(whole == 0.0, 0.0, e * far / whole)).sum(dim=1, keepdim=True).nan_to_num(0.0)
        self.relative = 3 * U * (far + mean_far) + (self.experts + 12) * U
        ids = torch.where(self.valid[:, None], chosen.cpu().long(), -1).flatten()
        self.counts = torch.bincount(ids[(ids >= 0) & (ids < self.experts)], minlength=self.experts).to(torch.int32)
        self.number = int(self.valid.sum())

    def loss(self):
        """loss, probabilities and the bounds on both: a column's sum takes at most 128 additions in 32 bits, then 64."""
        share = 1.0 / self.number if self.number else 0.0
        mean = self.p.sum(dim=0) * share
        off = (self.p * self.relative).sum(dim=0) * share + 130 * U * mean + 2.0 ** -120
        weight = self.coefficient * self.experts * self.counts.double() * share / self.choices
        value, bound = (weight * mean).sum().reshape(1), (weight.abs() * off).sum().reshape(1)
        return value, bound + 2 * U * value.abs(), mean, off + U * mean

    def gradient(self, upstream, dtype, counts=None, number=None, base=None):
        """The gradient and its bound, from counts of this call's own or given ones.

        An exp below 2^-126 that is taken as zero takes up to c 2^-126 from the row's sum of c p (1 / sum of exp <= 1), which p and the
        factor multiply: factor p 2^-126 sum c in all.  Each of the two products may end below 2^-126, where half a step is 2^-150; the
        second multiplies the first one's by |factor| at most."""
        c = (self.counts if counts is None else counts.cpu()[:self.experts]).double()
        number = self.number if number is None else number
        factor = upstream * self.coefficient * self.experts / self.choices / number ** 2 if number else 0.0
        dot = (self.p * c).sum(dim=1, keepdim=True)
        exact = factor * self.p * (c - dot)
        row = self.relative.amax(dim=1, keepdim=True)
        off_dot = (2 * row + (self.experts + 6) * U) * dot
        bound = abs(factor) * self.p * ((self.relative + 6 * U) * (c - dot).abs() + off_dot + 2 * U * c) + 2.0 ** -120 * abs(factor) * (c + dot)
        bound = bound + 2.0 ** -126 * abs(factor) * self.p * c.sum() + 2.0 ** -150 * (1.0 + abs(factor))
        exact, bound = torch.where(self.valid[:, None], exact, 0.0), torch.where(self.valid[:, None], bound, 0.0)
        if base is not None:
            exact = exact + base.cpu().double()
            bound = bound + U * exact.abs()
        return exact, bound + rounding(dtype, exact)
