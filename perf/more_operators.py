"""What the speed of the operators of a language model's training head is measured on: the
gradients of LayerNorm and RMSNorm (``layer_norm_bwd``, ``rms_norm_bwd``), and the cross entropy
of a projection onto a vocabulary without keeping its logits (``linear_cross_entropy_fwd``,
``linear_cross_entropy_bwd``).

A case is a dict of plain values.  Norms: ``op`` (ln_bwd, rms_bwd), ``rows``, ``cols``, ``dtype``,
``weight`` (its type).  Cross entropy: ``op`` (loss_fwd, loss_bwd), ``tokens``, ``hidden``,
``vocab``, ``dtype``, ``labels`` (their type), ``ignored`` (the share of tokens whose label does
not count), ``smoothing`` and ``z`` (the weight of the squared logsumexp).

``run`` computes the plain forms in 32 bits; where ``own`` is true it calls this package's
operators.  ``exact`` goes by the definition in 64 bits and takes the gradients of the norms by
automatic differentiation.
"""
import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16,
          "i32": torch.int32, "i64": torch.int64}
SIZES = {"fp32": 4, "fp16": 2, "bf16": 2, "i32": 4, "i64": 8}
EPS = 1e-5
IGNORED = -100
NORM = ("op", "rows", "cols", "dtype", "weight")
LOSS = ("op", "tokens", "hidden", "vocab", "dtype", "labels", "ignored", "smoothing", "z")
MOST_BYTES = 250_000_000  # of a drawn norm
MOST_FLOPS = 6e12         # of a drawn loss


def _case(name, *values):
    fields = NORM if values[0] in ("ln_bwd", "rms_bwd") else LOSS
    return {"name": name, **dict(zip(fields, values))}


def listed():
    return [
        # fine-tuning a small fp32 model on two short texts: latency
        _case("ln_small", "ln_bwd", 258, 768, "fp32", "fp32"),
        # one training step of 8192 tokens
        _case("ln_train", "ln_bwd", 8192, 4096, "bf16", "bf16"),
        # the widest rows of this repository's workloads, fp32 weights
        _case("ln_wide", "ln_bwd", 2048, 20480, "bf16", "fp32"),
        # the same step of a model with RMSNorm
        _case("rms_train", "rms_bwd", 8192, 4096, "bf16", "bf16"),
        # texts of ragged lengths, rows that are no whole number of 16 bytes
        _case("rms_ragged", "rms_bwd", 5003, 1001, "fp16", "fp32"),
        # the likelihood of the next token of four sequences: latency, the weights' read
        _case("loss_token", "loss_fwd", 4, 4096, 32000, "bf16", "i64", 0.0, 0.0, 0.0),
        # scoring candidate answers, an odd vocabulary, prompts ignored
        _case("loss_score", "loss_fwd", 1037, 2048, 50257, "fp16", "i32", 0.3, 0.0, 0.0),
        # one training step, a large vocabulary
        _case("loss_train", "loss_fwd", 8192, 4096, 128000, "bf16", "i64", 0.0, 0.0, 1e-4),
        # a small fp32 model
        _case("loss_small", "loss_fwd", 300, 768, 5003, "fp32", "i64", 0.1, 0.1, 0.0),
        # the gradients of a training step, the vocabulary of this repository's largest workload
        _case("grads_train", "loss_bwd", 8192, 4096, 32000, "bf16", "i64", 0.0, 0.0, 1e-4),
        # instruction tuning: only answers count
        _case("grads_tune", "loss_bwd", 2051, 2048, 50257, "bf16", "i64", 0.45, 0.1, 0.0),
        # a small fp32 model
        _case("grads_small", "loss_bwd", 257, 512, 8000, "fp32", "i64", 0.1, 0.0, 0.0),
    ]


def _log_uniform(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if rng.random() < 0.4:
        cols = int(_log_uniform(rng, 64, 32768))
        if rng.random() < 0.7:
            cols = max(64, cols // 64 * 64)
        rows = int(_log_uniform(rng, 1, 32768))
        weight = rng.choice([dtype, dtype, "fp32"])
        case = dict(zip(NORM, (rng.choice(["ln_bwd", "rms_bwd"]), rows, cols, dtype, weight)))
        while work(case)["bytes"] > MOST_BYTES:
            case["rows"] = case["rows"] * 2 // 3
        return case
    hidden = int(_log_uniform(rng, 128, 8192))
    if rng.random() < 0.85:
        hidden = max(128, hidden // 64 * 64)
    vocab = int(_log_uniform(rng, 1000, 160000))
    if rng.random() < 0.5:
        vocab = max(1024, vocab // 128 * 128)
    case = dict(zip(LOSS, (
        rng.choice(["loss_fwd", "loss_bwd"]), int(_log_uniform(rng, 1, 16384)), hidden, vocab,
        dtype, rng.choice(["i32", "i64"]), rng.choice([0.0, 0.0, rng.uniform(0.05, 0.7)]),
        rng.choice([0.0, 0.0, 0.1]), rng.choice([0.0, 0.0, 1e-4]))))
    while work(case)["flops"] > MOST_FLOPS:
        case["tokens"] = case["tokens"] * 2 // 3
    return case


def _live(case):
    """How many tokens count."""
    return case["tokens"] - round(case["ignored"] * case["tokens"])


def _randn(g, *shape):
    return torch.randn(*shape, device=DEVICE, generator=g)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    state = {"case": case}
    if "rows" in case:
        rows, cols = case["rows"], case["cols"]
        # a residual stream: channels of very different size, some off centre
        channel = torch.exp(0.5 * _randn(g, cols))
        state["x"] = (_randn(g, rows, cols) * channel + 0.3 * _randn(g, cols)).to(dtype)
        state["dy"] = _randn(g, rows, cols).to(dtype)
        state["weight"] = (1.0 + 0.2 * _randn(g, cols)).to(DTYPES[case["weight"]])
        state["bias"] = (0.1 * _randn(g, cols)).to(DTYPES[case["weight"]])
        return state
    tokens, hidden, vocab = case["tokens"], case["hidden"], case["vocab"]
    weight = (1.5 / math.sqrt(hidden) * _randn(g, vocab, hidden)).to(dtype)
    labels = torch.randint(0, vocab, (tokens,), device=DEVICE, generator=g)
    # a trained model: the label's logit stands out, more or less
    lean = 4.0 * torch.rand(tokens, 1, device=DEVICE, generator=g)
    x = (_randn(g, tokens, hidden) + lean * weight[labels].float()).to(dtype)
    order = torch.randperm(tokens, device=DEVICE, generator=g)
    labels[order[_live(case):]] = IGNORED
    state.update(x=x, weight=weight, labels=labels.to(DTYPES[case["labels"]]))
    if case["op"] == "loss_bwd":
        w = weight.float()
        state["lse"] = torch.cat([torch.logsumexp(part.float() @ w.T, 1) for part in x.split(2048)])
        # of the mean loss, scaled up where the type's range is small
        mean = (4096.0 if case["dtype"] == "fp16" else 1.0) / max(1, _live(case))
        state["dloss"] = torch.full((tokens,), mean, device=DEVICE)
    return state


def _plain_norm(state):
    case = state["case"]
    x, dy, w = (state[n].float() for n in ("x", "dy", "weight"))
    if case["op"] == "ln_bwd":
        x = x - x.mean(1, keepdim=True)
    size = torch.rsqrt((x * x).mean(1, keepdim=True) + EPS)
    unit, du = x * size, dy * w
    dx = du - unit * (du * unit).mean(1, keepdim=True)
    wtype = DTYPES[case["weight"]]
    out = [(dy * unit).sum(0).to(wtype)]
    if case["op"] == "ln_bwd":
        dx = dx - du.mean(1, keepdim=True)
        out.append(dy.sum(0).to(wtype))
    return [(size * dx).to(DTYPES[case["dtype"]])] + out


def _plain_loss(state):
    case = state["case"]
    x, w = state["x"].float(), state["weight"].float()
    labels = state["labels"].long()
    counts = (labels != IGNORED)[:, None]
    at = labels.clamp(min=0)[:, None]
    logits = x @ w.T
    s, z, vocab = case["smoothing"], case["z"], case["vocab"]
    if case["op"] == "loss_fwd":
        most = logits.max(1, keepdim=True).values
        lse = (logits - most).exp().sum(1, keepdim=True).log() + most
        loss = lse - (1.0 - s) * logits.gather(1, at)
        if s:
            loss = loss - s / vocab * logits.sum(1, keepdim=True)
        square = z * lse * lse
        return [torch.where(counts, t, 0.0)[:, 0] for t in (loss + square, lse, square)]
    lse = state["lse"][:, None]
    p = (logits - lse).exp() * (1.0 + 2.0 * z * lse)
    if s:
        p = p - s / vocab
    p.scatter_add_(1, at, torch.full_like(lse, s - 1.0))
    p = torch.where(counts, p * state["dloss"][:, None], 0.0)
    dtype = DTYPES[case["dtype"]]
    return [(p @ w).to(dtype), (p.T @ x).to(dtype)]


def _own(state):
    case = state["case"]
    if case["op"] == "ln_bwd":
        from dslperfgap_amd.viperbench.layer_norm.hip_impl import layer_norm_bwd
        return layer_norm_bwd(state["dy"], state["x"], state["weight"], state["bias"], EPS)
    if case["op"] == "rms_bwd":
        from dslperfgap_amd.viperbench.rms_norm.hip_impl import rms_norm_bwd
        return rms_norm_bwd(state["dy"], state["x"], (case["cols"],), state["weight"], EPS)
    from dslperfgap_amd.viperbench.linear_cross_entropy.hip_impl import (linear_cross_entropy_bwd,
                                                                         linear_cross_entropy_fwd)
    how = {"smoothing": case["smoothing"], "lse_square_scale": case["z"],
           "ignored_index": IGNORED}
    if case["op"] == "loss_fwd":
        return linear_cross_entropy_fwd(state["x"], state["weight"], state["labels"], **how)
    return linear_cross_entropy_bwd(state["dloss"], state["x"], state["weight"], state["lse"],
                                    state["labels"], **how)


def run(state):
    if own:
        return list(_own(state))
    return _plain_norm(state) if "rows" in state["case"] else _plain_loss(state)


def work(case):
    e = SIZES[case["dtype"]]
    if "rows" in case:
        n, vectors = case["rows"] * case["cols"], 4 if case["op"] == "ln_bwd" else 2
        return {"bytes": 3 * n * e + (vectors - 1) * case["cols"] * SIZES[case["weight"]],
                "flops": (16 if case["op"] == "ln_bwd" else 11) * n}
    live, tokens = _live(case), case["tokens"]
    weight = case["vocab"] * case["hidden"] * e
    product = 2 * live * case["hidden"] * case["vocab"]
    if case["op"] == "loss_fwd":
        return {"bytes": live * case["hidden"] * e + weight + tokens * (SIZES[case["labels"]] + 12),
                "flops": product}
    return {"bytes": (live + tokens) * case["hidden"] * e + 2 * weight +
            tokens * (SIZES[case["labels"]] + 8), "flops": 3 * product}


def exact(case, seed):
    state = prepare(case, seed)
    if "rows" in case:
        leaves = [state[n].double().requires_grad_() for n in ("x", "weight", "bias")]
        with torch.enable_grad():
            x, w, b = leaves
            if case["op"] == "ln_bwd":
                var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
                y = (x - mean) / (var + EPS).sqrt() * w + b
            else:
                y = x / (x.square().sum(1, keepdim=True) / case["cols"] + EPS).sqrt() * w
                leaves = leaves[:2]
            return list(torch.autograd.grad(y, leaves, state["dy"].double()))
    labels = state["labels"].long()
    keep = (labels != IGNORED).nonzero()[:, 0]
    x, w = state["x"].double(), state["weight"].double()
    s, z, vocab = case["smoothing"], case["z"], case["vocab"]
    parts = []
    dw = torch.zeros_like(w)
    dx = torch.zeros_like(x)
    for rows in keep.split(2048):
        logits = torch.matmul(x[rows], w.T)
        target = torch.full_like(logits, s / vocab)
        target[torch.arange(len(rows), device=DEVICE), labels[rows]] += 1.0 - s
        if case["op"] == "loss_fwd":
            lse = torch.logsumexp(logits, 1)
            square = z * lse * lse
            parts.append(torch.stack([lse - (target * logits).sum(1) + square, lse, square]))
            continue
        lse = state["lse"][rows].double()[:, None]
        d = torch.exp(logits - lse) * (1.0 + 2.0 * z * lse) - target
        d *= state["dloss"][rows].double()[:, None]
        dx[rows] = torch.matmul(d, w)
        dw += torch.matmul(d.T, x[rows])
    if case["op"] == "loss_bwd":
        return [dx, dw]
    out = torch.zeros(3, case["tokens"], dtype=torch.float64, device=DEVICE)
    if parts:
        out[:, keep] = torch.cat(parts, 1)
    return list(out)
