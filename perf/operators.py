"""What the operators of a language model's training step are timed on, in plain torch and through the framework.

Three families, each beside a primitive of the framework: the embedding lookup and its gradient (sorted pairs), the norm
of all gradients and their clipping (reduction over a list of views), and the balance loss of a router with the counts
per expert and its gradient (histogram).

With `own` false `run` computes each operator with elementary torch operations in 32 bits (long sums in 64), rounded
once; with `own` true it makes the calls that a program makes of the framework.
"""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "int32": torch.int32, "int64": torch.int64}


def listed():
    return [
        # one token for each of eight sequences: a decoding step
        {"name": "lookup_decode", "op": "lookup", "tokens": 8, "rows": 32_000, "width": 4_096, "type": "bf16", "out": "bf16", "ids": "int64",
         "scale": 64.0, "padded": 0.0},
        # the tokens of a batch of long sequences, the ends of some of them padded with -1
        {"name": "lookup_batch", "op": "lookup", "tokens": 65_536, "rows": 128_000, "width": 4_096, "type": "bf16", "out": "bf16", "ids": "int32",
         "scale": 1.0, "padded": 0.05},
        # a short sequence and a small 32-bit model
        {"name": "gradient_short", "op": "gradient", "tokens": 301, "rows": 10_007, "width": 768, "type": "fp32", "out": "fp32", "ids": "int64",
         "scale": 27.7, "padded": 0.0},
        # an ordinary batch of one GPU: 16-bit activations, gradients held in 32 bits
        {"name": "gradient_batch", "op": "gradient", "tokens": 16_384, "rows": 32_000, "width": 2_048, "type": "bf16", "out": "fp32", "ids": "int64",
         "scale": 1.0, "padded": 0.0},
        # a large batch into a large vocabulary
        {"name": "gradient_large", "op": "gradient", "tokens": 131_072, "rows": 128_000, "width": 4_096, "type": "bf16", "out": "fp32", "ids": "int32",
         "scale": 1.0, "padded": 0.05},
        # a small model's few tensors, where launches are what costs
        {"name": "clip_small", "op": "clip", "tensors": 14, "elements": 300_000, "type": "fp32", "out": "fp32", "packed": False, "max_norm": 1.0},
        # the shard of a model that one GPU holds: a few hundred tensors, matrices beside short vectors
        {"name": "clip_shard", "op": "clip", "tensors": 219, "elements": 60_000_000, "type": "bf16", "out": "bf16", "packed": False, "max_norm": 1.0},
        # the norm alone, for a log or for a sum over ranks, of a billion gradients in 32 bits packed one behind the other
        {"name": "norm_large", "op": "norm", "tensors": 291, "elements": 1_000_000_000, "type": "fp32", "packed": True},
        # a router of few experts and a handful of tokens
        {"name": "balance_small", "op": "balance", "tokens": 64, "experts": 8, "choices": 2, "type": "fp32", "ids": "int64", "padded": 0.0},
        # many tokens of a padded batch, 16-bit logits
        {"name": "balance_large", "op": "balance", "tokens": 262_144, "experts": 128, "choices": 8, "type": "bf16", "ids": "int32", "padded": 0.1},
        # its gradient for an odd number of experts and tokens
        {"name": "balance_gradient_ragged", "op": "balance_gradient", "tokens": 8_191, "experts": 60, "choices": 4, "type": "fp32", "ids": "int64",
         "padded": 0.0},
        # and for many experts
        {"name": "balance_gradient_large", "op": "balance_gradient", "tokens": 131_072, "experts": 256, "choices": 8, "type": "fp32", "ids": "int64",
         "padded": 0.1},
    ]


def _size(rng, least, most):
    return int(math.exp(rng.uniform(math.log(least), math.log(most + 1))))


def draw(rng):
    op = rng.choice(["lookup", "gradient", "gradient", "clip", "clip", "norm", "balance", "balance_gradient"])
    kind = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    ids, padded = rng.choice(["int32", "int64"]), rng.choice([0.0, 0.0, 0.1])
    if op in ("lookup", "gradient"):
        width = _size(rng, 64, 8_192)
        if rng.random() < 0.7:  # widths of models are multiples of powers of two; some are not
            width = max(64, width // 64 * 64)
        rows = _size(rng, 500, min(128_000, (1 << 29) // width))
        tokens = _size(rng, 1, min(131_072, (1 << 28) // width))
        out = rng.choice([kind, "fp32" if op == "gradient" else "bf16"])
        return {"op": op, "tokens": tokens, "rows": rows, "width": width, "type": kind, "out": out, "ids": ids,
                "scale": rng.choice([1.0, round(math.sqrt(width), 3)]), "padded": padded}
    if op in ("clip", "norm"):
        case = {"op": op, "tensors": _size(rng, 1, 1_500), "elements": _size(rng, 20_000, 400_000_000), "type": kind, "packed": rng.random() < 0.3}
        if op == "clip":  # most steps are clipped at the start of a training, few later on
            case |= {"out": rng.choice([kind, kind, "bf16"]), "max_norm": rng.choice([1.0, 1.0, 1e6])}
        return case
    experts = _size(rng, 4, 512)
    choices = rng.randint(1, min(8, experts))
    return {"op": op, "tokens": _size(rng, 1, min(262_144, (1 << 25) // experts)), "experts": experts, "choices": choices, "type": kind, "ids": ids,
            "padded": padded}


# ---- inputs --------------------------------------------------------------------------------------
COEFFICIENT = 0.01


def _frequencies(rows):
    """How often each token comes: falling as a power of its rank, as words do."""
    return torch.arange(1, rows + 1, dtype=torch.float64).pow(-1.0).div_(math.log(rows) + 0.5772)


def _tokens(case, gen):
    """Tokens by their frequency (the inverse of its running sum), ranks scattered over the vocabulary; the padded ones are -1."""
    rows, n = case["rows"], case["tokens"]
    ends = _frequencies(rows).cumsum(0).cuda()
    rank = torch.searchsorted(ends, torch.rand(n, generator=gen, device="cuda", dtype=torch.float64) * ends[-1]).clamp_(max=rows - 1)
    tokens = torch.randperm(rows, generator=gen, device="cuda")[rank]
    if case["padded"]:
        tokens[n - int(n * case["padded"]):] = -1
    return tokens.to(TYPES[case["ids"]])


def _lengths(case):
    """Lengths of a model's tensors: a few orders of magnitude apart, together about `elements`."""
    rng = random.Random(case["tensors"] * 1_000_003 + case["elements"])
    shares = [math.exp(rng.uniform(0.0, 9.0)) for _ in range(case["tensors"])]
    whole = sum(shares)
    return [max(1, int(case["elements"] * s / whole)) for s in shares]


def _places(case):
    """Where each tensor begins in the buffer: packed one behind the other, or each on a boundary of 128 elements."""
    at, places = 0, []
    for n in _lengths(case):
        places.append(at)
        at += n if case["packed"] else -(-n // 128) * 128
    return places, at


def _router(case, gen):
    t, e, k = case["tokens"], case["experts"], case["choices"]
    # experts differ in how well liked they are; tokens choose by the logits that the loss sees
    logits = torch.randn(t, e, generator=gen, device="cuda") * 1.5 + torch.randn(e, generator=gen, device="cuda")
    chosen = logits.topk(k, dim=1).indices.to(TYPES[case["ids"]])
    mask = None
    if case["padded"]:
        mask = torch.ones(t, dtype=torch.bool, device="cuda")
        mask[t - int(t * case["padded"]):] = False
    return logits.to(TYPES[case["type"]]), chosen.contiguous(), mask


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op == "lookup":
        table = torch.empty(case["rows"], case["width"], dtype=TYPES[case["type"]], device="cuda").normal_(0.0, 0.02, generator=gen)
        return {"table": table, "tokens": _tokens(case, gen)}
    if op == "gradient":
        upstream = torch.empty(case["tokens"], case["width"], dtype=TYPES[case["type"]], device="cuda").normal_(0.0, 0.01, generator=gen)
        return {"tokens": _tokens(case, gen), "upstream": upstream}
    if op in ("clip", "norm"):
        places, whole = _places(case)
        flat = torch.zeros(whole, dtype=TYPES[case["type"]], device="cuda")
        sizes = torch.rand(len(places), generator=gen, device="cuda").mul_(-3.0).exp_().tolist()  # layers differ in how large their gradients are
        views = [flat[at:at + n] for at, n in zip(places, _lengths(case))]
        for view, size in zip(views, sizes):
            view.normal_(0.0, 0.02 * size, generator=gen)
        return {"flat": flat, "views": views}
    logits, chosen, mask = _router(case, gen)
    inputs = {"logits": logits, "chosen": chosen, "mask": mask}
    if op == "balance_gradient":
        inputs["counts"] = _counts(chosen, mask, case["experts"])
        # training in fp16 scales its loss until the gradients, one token's share of a mean, lie in the type's range
        inputs["loss_gradient"] = (torch.rand(1, generator=gen, device="cuda") + 0.5) * (64.0 * case["tokens"] if case["type"] == "fp16" else 1.0)
    return inputs


def _counts(chosen, mask, experts):
    """How often each expert is chosen by a token that counts, and behind them the number of these tokens."""
    tokens = chosen.shape[0]
    valid = torch.ones(tokens, dtype=torch.bool, device=chosen.device) if mask is None else mask
    slots = torch.where(valid[:, None], chosen.long(), experts).reshape(-1)
    counts = torch.zeros(experts + 1, dtype=torch.int32, device=chosen.device)
    counts.index_add_(0, slots, torch.ones_like(slots, dtype=torch.int32))
    counts[experts] = valid.sum()
    return counts


def prepare(case, seed):
    state = {"case": case} | _inputs(case, seed)
    if own:
        state |= _handles(case, state)
    return state


def _handles(case, state):
    """What a program that uses the framework keeps beside its data: the calls, workspaces and the buffers that receive the results."""
    import ilgpu_b200 as ib

    acc = ib.Accelerator(0)
    op = case["op"]
    if op == "lookup":
        return {"call": acc.CreateEmbedding(), "result": torch.empty(case["tokens"], case["width"], dtype=TYPES[case["out"]], device="cuda")}
    if op == "gradient":
        ints = acc.ComputeEmbeddingGradientTempStorageSize(case["rows"], case["width"], case["tokens"])
        return {"call": acc.CreateEmbeddingGradient(), "temp": acc.Allocate1D(ints, torch.int32),
                "result": torch.empty(case["rows"], case["width"], dtype=TYPES[case["out"]], device="cuda")}
    if op in ("clip", "norm"):
        temp = acc.Allocate1D(acc.ComputeGradientNormTempStorageSize(case["tensors"]), torch.int32)
        handles = {"temp": temp, "norm": torch.empty(1, device="cuda")}
        if op == "norm":
            return handles | {"call": acc.CreateGradientNorm()}
        result = torch.zeros(state["flat"].numel(), dtype=TYPES[case["out"]], device="cuda")
        outputs = [result[at:at + n] for at, n in zip(_places(case)[0], _lengths(case))]
        return handles | {"call": acc.CreateGradientClip(), "result": result, "outputs": outputs}
    if op == "balance":
        ints = acc.ComputeBalanceLossTempStorageSize(case["experts"], case["tokens"])
        return {"call": acc.CreateBalanceLoss(COEFFICIENT), "temp": acc.Allocate1D(ints, torch.int32), "loss": torch.empty(1, device="cuda"),
                "counts": torch.empty(case["experts"] + 1, dtype=torch.int32, device="cuda"), "probabilities": torch.empty(case["experts"], device="cuda")}
    return {"call": acc.CreateBalanceLossGradient(COEFFICIENT, case["choices"]), "result": torch.empty_like(state["logits"])}


# ---- one pass ------------------------------------------------------------------------------------
def run(state):
    case, op = state["case"], state["case"]["op"]
    if own:
        return _run_own(state, case, op)
    if op == "lookup":
        return _lookup(state["table"], state["tokens"], case["scale"], TYPES[case["out"]])
    if op == "gradient":
        return _gradient(state["tokens"], state["upstream"], case["rows"], case["scale"], TYPES[case["out"]])
    if op == "norm":
        return {"norm": _norm(state["flat"])}
    if op == "clip":
        norm = _norm(state["flat"])
        factor = torch.where(norm > case["max_norm"], case["max_norm"] / norm, torch.ones_like(norm))
        return {"norm": norm, "clipped": (state["flat"].float() * factor).to(TYPES[case["out"]])}
    if op == "balance":
        return _balance(state["logits"], state["chosen"], state["mask"])
    return _balance_gradient(state["logits"], state["mask"], state["counts"], state["loss_gradient"], case["choices"])


def _run_own(state, case, op):
    call = state["call"]
    if op == "lookup":
        call(None, state["table"], state["tokens"], state["result"], case["scale"])
        return state["result"]
    if op == "gradient":
        call(None, state["tokens"], state["upstream"], state["result"], state["temp"], case["scale"])
        return state["result"]
    if op == "norm":
        call(None, state["views"], state["norm"], state["temp"])
        return {"norm": state["norm"]}
    if op == "clip":
        call(None, state["views"], state["outputs"], case["max_norm"], state["norm"], state["temp"])
        return {"norm": state["norm"], "clipped": state["result"]}
    if op == "balance":
        call(None, state["logits"], state["chosen"], state["mask"], state["loss"], state["counts"], state["probabilities"], state["temp"])
        return {"loss": state["loss"], "counts": state["counts"], "probabilities": state["probabilities"]}
    call(None, state["logits"], state["mask"], state["counts"], state["loss_gradient"], state["result"])
    return state["result"]


# ---- the operators in their plain form -------------------------------------------------------------
def _lookup(table, tokens, scale, dtype):
    there = (tokens >= 0) & (tokens < table.shape[0])
    rows = table[torch.where(there, tokens, 0)].float() * scale
    return torch.where(there[:, None], rows, 0.0).to(dtype)


def _gradient(tokens, upstream, rows, scale, dtype):
    there = (tokens >= 0) & (tokens < rows)
    anywhere = torch.arange(tokens.shape[0], device=tokens.device, dtype=tokens.dtype) % rows  # where the zeros of padded tokens go
    sums = torch.zeros(rows, upstream.shape[1], device=upstream.device)
    sums.index_add_(0, torch.where(there, tokens, anywhere), torch.where(there[:, None], upstream.float(), 0.0))
    return (sums * scale).to(dtype)


def _norm(flat):
    return flat.float().square().sum(dtype=torch.float64).sqrt().float().reshape(1)


def _softmax(logits):
    x = logits.float()
    top = x.amax(dim=1, keepdim=True)
    e = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    whole = e.sum(dim=1, keepdim=True)
    return torch.where(whole == 0.0, 0.0, e / whole)


def _balance(logits, chosen, mask):
    experts, choices = logits.shape[1], chosen.shape[1]
    counts = _counts(chosen, mask, experts)
    p = _softmax(logits)
    if mask is not None:
        p = torch.where(mask[:, None], p, 0.0)
    tokens = counts[experts].double()
    inverse = torch.where(tokens > 0, 1.0 / tokens, 0.0)
    mean = p.sum(dim=0, dtype=torch.float64) * inverse
    loss = COEFFICIENT * experts * (counts[:experts].double() * inverse / choices * mean).sum()
    return {"loss": loss.float().reshape(1), "counts": counts, "probabilities": mean.float()}


def _balance_gradient(logits, mask, counts, loss_gradient, choices):
    experts = logits.shape[1]
    p = _softmax(logits)
    often = counts[:experts].float()
    tokens = counts[experts].double()
    factor = torch.where(tokens > 0, loss_gradient * (COEFFICIENT * experts / choices) / (tokens * tokens), 0.0).float()
    gradient = factor * p * (often - (p * often).sum(dim=1, keepdim=True))
    if mask is not None:
        gradient = torch.where(mask[:, None], gradient, 0.0)
    return gradient.to(logits.dtype)


# ---- from the definitions in 64 bits ---------------------------------------------------------------
def exact(case, seed):
    inputs = _inputs(case, seed)
    op = case["op"]
    if op == "lookup":
        result = torch.zeros(case["tokens"], case["width"], dtype=torch.float64, device="cuda")
        at = (inputs["tokens"] >= 0).nonzero().reshape(-1)
        result[at] = inputs["table"].index_select(0, inputs["tokens"][at].long()).double() * case["scale"]
        return result
    if op == "gradient":
        result = torch.zeros(case["rows"], case["width"], dtype=torch.float64, device="cuda")
        at = (inputs["tokens"] >= 0).nonzero().reshape(-1)
        for some in at.split(8_192):  # sums of a part of the tokens at a time
            result.index_put_((inputs["tokens"][some].long(),), inputs["upstream"][some].double() * case["scale"], accumulate=True)
        return result
    if op in ("clip", "norm"):
        norm = math.sqrt(math.fsum(float(part.double().pow(2).sum()) for part in inputs["flat"].split(1 << 26)))
        whole = torch.tensor([norm], dtype=torch.float64, device="cuda")
        return {"norm": whole} if op == "norm" else {"norm": whole, "clipped": inputs["flat"].double() * min(1.0, case["max_norm"] / norm)}
    x, experts, choices = inputs["logits"].double(), case["experts"], case["choices"]
    p = (x - x.logsumexp(dim=1, keepdim=True)).exp()
    valid = torch.ones(case["tokens"], dtype=torch.float64, device="cuda") if inputs["mask"] is None else inputs["mask"].double()
    tokens = max(1.0, float(valid.sum()))
    often = torch.stack([((inputs["chosen"] == e).sum(dim=1) * valid).sum() for e in range(experts)])
    if op == "balance":
        mean = (p * valid[:, None]).sum(dim=0) / tokens
        counts = torch.cat([often, valid.sum().reshape(1)]).round().to(torch.int32)
        return {"loss": (COEFFICIENT * experts * (often / (tokens * choices) * mean).sum()).reshape(1), "counts": counts, "probabilities": mean}
    # the derivative of the loss in each logit, of one softmax: diag(p) - p p'
    slope = COEFFICIENT * experts * often / (tokens * choices) / tokens * inputs["loss_gradient"].double()
    return valid[:, None] * (p * slope - p * (p @ slope[:, None]))


# ---- what a pass cannot do without -----------------------------------------------------------------
def work(case):
    op, size = case["op"], TYPES[case["type"]].itemsize
    if op == "lookup":
        n = case["tokens"] - int(case["tokens"] * case["padded"])
        distinct = float((1.0 - (1.0 - _frequencies(case["rows"]).clamp(max=1.0)).pow(n)).sum())  # each row is read once
        cells = case["tokens"] * case["width"]
        return {"bytes": distinct * case["width"] * size + cells * TYPES[case["out"]].itemsize + case["tokens"] * TYPES[case["ids"]].itemsize,
                "flops": cells}
    if op == "gradient":
        n = case["tokens"] - int(case["tokens"] * case["padded"])
        return {"bytes": n * case["width"] * size + case["rows"] * case["width"] * TYPES[case["out"]].itemsize
                + case["tokens"] * TYPES[case["ids"]].itemsize, "flops": n * case["width"]}
    if op in ("clip", "norm"):
        n = sum(_lengths(case))
        return {"bytes": n * (size + (TYPES[case["out"]].itemsize if op == "clip" else 0)), "flops": n * (3 if op == "clip" else 2)}
    n = case["tokens"] - int(case["tokens"] * case["padded"])
    cells, ids = n * case["experts"], n * case["choices"] * TYPES[case["ids"]].itemsize
    if op == "balance":
        return {"bytes": cells * size + ids + case["experts"] * 8, "flops": cells * 5}
    return {"bytes": (cells + case["tokens"] * case["experts"]) * size + case["experts"] * 4, "flops": cells * 8}
