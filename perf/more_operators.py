"""Timed cases of the operators of a model's blocks and head, ``minispeed_amd.ops``.

Three operators of a training step, each in its directions:

``loss``, ``loss_grad``
    log probabilities of given tokens under a large vocabulary, straight from the
    hidden states and the head's weight, without keeping the logits; and the
    gradients of both
``norm``, ``norm_grad``
    what lies between two blocks of a model: the norm after the one, its gate and
    residual scale, the residual sum and the norm before the next; and all of
    their gradients
``bias``, ``bias_grad``
    the learned relative position bias of attention, a table over buckets of
    distances; and the gradient of the table

A case names the operator, its sizes, its element type and what its inputs are
like.  Outputs come whole.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}
IGNORE = -100
EPS = 1e-5
LOSS_OPS = ("loss", "loss_grad")
NORM_OPS = ("norm", "norm_grad")
BIAS_OPS = ("bias", "bias_grad")


def listed():
    return [
        # the tiny GPT's head (8 x 128 tokens, width 256, vocab 512): latency counts
        dict(name="loss-tiny", op="loss", rows=1024, width=256, vocab=512, dtype="fp32",
             ignored=0.0),
        # scoring the next token of four sequences with the 8B decoder's head:
        # reading the weight is all there is
        dict(name="loss-few", op="loss", rows=4, width=4096, vocab=128256, dtype="bf16",
             ignored=0.0),
        # the loss of 4 x 2048 tokens of the 1.3B GPT
        dict(name="loss-1.3b", op="loss", rows=8192, width=2048, vocab=50257, dtype="fp16",
             ignored=0.1),
        # the backward pass of 16 x 1024 tokens of the 124M GPT, prompts left out
        dict(name="loss-grad-124m", op="loss_grad", rows=16384, width=768, vocab=50257,
             dtype="bf16", ignored=0.1),
        # the backward pass of 2048 tokens of the 8B decoder
        dict(name="loss-grad-8b", op="loss_grad", rows=2048, width=4096, vocab=128256,
             dtype="bf16", ignored=0.0),
        # between two half-blocks of the tiny GPT
        dict(name="norm-tiny", op="norm", rows=1024, width=256, groups=0, dtype="fp32",
             kind="layer", post=False, scale=1.0),
        # between two half-blocks of the 1.3B GPT, 4 x 2048 tokens
        dict(name="norm-1.3b", op="norm", rows=8192, width=2048, groups=0, dtype="fp16",
             kind="layer", post=False, scale=1.0),
        # the same of the 124M GPT with a gate for each of 16 sequences, backward
        dict(name="norm-grad-124m", op="norm_grad", rows=16384, width=768, groups=16,
             dtype="bf16", kind="layer", post=False, scale=1.0),
        # 8192 tokens of the 8B decoder's width: norms on both sides of the block,
        # a gate for each channel and a residual scale, backward
        dict(name="norm-grad-8b", op="norm_grad", rows=8192, width=4096, groups=1,
             dtype="bf16", kind="rms", post=True, scale=0.5),
        # one new token of the 8B decoder's 32 heads after a cache of 4096
        dict(name="bias-token", op="bias", heads=32, batch=1, queries=1, keys=4097, buckets=32,
             distance=128, causal=True, dtype="bf16"),
        # 16 heads over 2048 tokens of the 1.3B GPT
        dict(name="bias-1.3b", op="bias", heads=16, batch=1, queries=2048, keys=2048, buckets=32,
             distance=128, causal=True, dtype="fp16"),
        # 8 sequences of 1024 tokens of the 124M GPT's 12 heads share the table
        dict(name="bias-grad-124m", op="bias_grad", heads=12, batch=8, queries=1024, keys=1024,
             buckets=64, distance=256, causal=False, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, hi):
    width = _log_int(rng, 64, hi)
    return max(64, width // 64 * 64) if rng.random() < 0.75 else width


def draw(rng):
    op = rng.choice(LOSS_OPS + NORM_OPS + BIAS_OPS)
    dtype = rng.choice(("fp32", "fp16", "bf16"))
    if op in LOSS_OPS:
        width, vocab, rows = _width(rng, 4096), _log_int(rng, 512, 128256), _log_int(rng, 1, 16384)
        # 32 bits cost several times the products of 16
        most = 1.8e11 if dtype == "fp32" else 1.07e12
        while rows * width * vocab > most or rows * vocab > 8.3e8:
            rows = max(1, rows // 2)
        return dict(op=op, rows=rows, width=width, vocab=vocab, dtype=dtype,
                    ignored=rng.choice((0.0, 0.1, 0.5)))
    if op in NORM_OPS:
        width, rows = _width(rng, 16384), _log_int(rng, 1, 16384)
        while rows * width * BYTES[dtype] > 6.7e7:
            rows = max(1, rows // 2)
        gate = rng.choice(("none", "channel", "sequence", "token"))
        groups = {"none": 0, "channel": 1, "token": rows}.get(gate)
        if groups is None:
            groups = max(k for k in range(1, 17) if rows % k == 0)
        return dict(op=op, rows=rows, width=width, groups=groups, dtype=dtype,
                    kind=rng.choice(("rms", "layer")), post=rng.random() < 0.5,
                    scale=rng.choice((1.0, 0.5, 1.7)))
    heads, batch = _log_int(rng, 1, 32), _log_int(rng, 1, 8) if op == "bias_grad" else 1
    keys = _log_int(rng, 1, 8192)
    queries = rng.choice((1, keys, _log_int(rng, 1, keys)))
    while heads * batch * queries * keys * BYTES[dtype] > 2e8:
        batch, heads = max(1, batch // 2), max(1, heads // 2) if batch == 1 else heads
        if batch == heads == 1:
            break
    buckets = rng.choice((8, 32, 64, 128))
    return dict(op=op, heads=heads, batch=batch, queries=queries, keys=keys, buckets=buckets,
                distance=buckets * rng.choice((2, 4, 16)) + rng.choice((0, 1)),
                causal=rng.random() < 0.5, dtype=dtype)


# -- inputs -----------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt, op = DTYPES[case["dtype"]], case["op"]

    def randn(*shape, std=1.0, mean=0.0):
        x = torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)
        return x.mul_(std).add_(mean).to(dt)

    if op in LOSS_OPS:
        n, d, v = case["rows"], case["width"], case["vocab"]
        weight = randn(v, d, std=0.02)
        targets = torch.randint(0, v, (n,), generator=g, device="cuda")
        # hidden states behind a norm that lean towards the given token, as in a trained model
        lean = 6.0 / (0.02 * 0.02 * d)
        hidden = (torch.randn(n, d, generator=g, device="cuda")
                  + lean * weight[targets].float()).to(dt)
        if case["ignored"]:
            out = torch.rand(n, generator=g, device="cuda") < case["ignored"]
            targets = torch.where(out, torch.full_like(targets, IGNORE), targets)
        st = {"case": case, "hidden": hidden, "weight": weight, "targets": targets}
        if op == "loss_grad":
            # what the forward pass left, and the gradients that come down: of a
            # mean over the tokens with some weighting, and of a penalty on lse
            st["lse"] = torch.cat([torch.logsumexp(h.float() @ weight.float().T, 1)
                                   for h in hidden.split(2048)])
            st["grad_logprob"] = (torch.randn(n, generator=g, device="cuda") * 0.1 - 1.0) / n
            st["grad_lse"] = st["lse"] * (2e-4 / n)
        return st

    if op in NORM_OPS:
        n, w, groups = case["rows"], case["width"], case["groups"]
        # a residual stream with some channels far larger than the others
        spread = torch.exp(torch.randn(w, generator=g, device="cuda") * 0.7)
        residual = (torch.randn(n, w, generator=g, device="cuda") * spread + 0.1 * spread).to(dt)
        st = {"case": case, "block": randn(n, w, std=0.7), "weight": randn(w, std=0.1, mean=1.0),
              "bias": randn(w, std=0.1) if case["kind"] == "layer" else None,
              "block_weight": randn(w, std=0.1, mean=1.0) if case["post"] else None,
              "block_bias": randn(w, std=0.1) if case["post"] and case["kind"] == "layer" else None,
              "gate": randn(groups, w, std=0.3, mean=0.5) if groups else None}
        if groups:
            # rows in groups, each with a gate of its own
            st["block"] = st["block"].view(groups, n // groups, w)
            residual = residual.view(groups, n // groups, w)
            st["gate"] = st["gate"].view(groups, 1, w) if groups > 1 else st["gate"].view(w)
        st["residual"] = residual
        if op == "norm_grad":
            # the residual and the statistics that the forward pass left, in place of
            # the residual before the block
            stats = list(_stats(residual.double(), case["kind"]))
            if case["post"]:
                stats += _stats(st["block"].double(), case["kind"])
            st["stats"] = torch.cat(stats, -1).float()
            shape = residual.shape
            st["grad_out"] = randn(*shape, std=1e-2)
            st["grad_residual"] = randn(*shape, std=1e-2)
        return st

    h, b = case["heads"], case["buckets"]
    if op == "bias":
        return {"case": case, "table": randn(b, h, std=0.5)}
    return {"case": case, "grad": randn(case["batch"], h, case["queries"], case["keys"], std=1e-3)}


def _stats(x, kind):
    """Mean and reciprocal deviation of the last dimension (the mean of ``rms`` is 0)."""
    mean = x.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(x[..., :1])
    return mean, ((x - mean).square().mean(-1, keepdim=True) + EPS).rsqrt()


# -- one pass ---------------------------------------------------------------

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(st):
    import minispeed_amd as ms
    ops, case = ms.ops, st["case"]
    op = case["op"]
    if op == "loss":
        r = ops.linear_logprobs(st["hidden"], st["weight"], st["targets"], ignore_index=IGNORE)
        return {"logprob": r.logprob, "lse": r.lse}
    if op == "loss_grad":
        dh, dw = ops.linear_logprobs_grad(st["hidden"], st["weight"], st["targets"], st["lse"],
                                          st["grad_logprob"], st["grad_lse"], ignore_index=IGNORE)
        return {"hidden": dh, "weight": dw}
    if op == "norm":
        r = ops.residual_norm(st["residual"], st["block"], st["weight"], bias=st["bias"],
                              block_weight=st["block_weight"], block_bias=st["block_bias"],
                              gate=st["gate"], scale=case["scale"], eps=EPS, kind=case["kind"])
        return {"residual": r.residual, "out": r.out}
    if op == "norm_grad":
        r = ops.residual_norm_grad(st["grad_out"], st["grad_residual"], st["residual"],
                                   st["stats"], st["block"], st["weight"], bias=st["bias"],
                                   block_weight=st["block_weight"], block_bias=st["block_bias"],
                                   gate=st["gate"], scale=case["scale"], kind=case["kind"])
        return {k: v for k, v in r._asdict().items() if v is not None}
    if op == "bias":
        return ops.position_bias(st["table"], case["queries"], case["keys"],
                                 max_distance=case["distance"], causal=case["causal"])
    return ops.position_bias_grad(st["grad"], case["buckets"], max_distance=case["distance"],
                                  causal=case["causal"])


def _run_plain(st):
    case = st["case"]
    op, dt = case["op"], DTYPES[case["dtype"]]
    if op in LOSS_OPS:
        h, w, targets = st["hidden"].float(), st["weight"].float(), st["targets"]
        given = targets != IGNORE
        at = targets.clamp(min=0)[:, None]
        x = h @ w.T
    if op == "loss":
        most = x.amax(1, keepdim=True)
        lse = (most + torch.log(torch.exp(x - most).sum(1, keepdim=True)))[:, 0]
        return {"logprob": torch.where(given, x.gather(1, at)[:, 0] - lse, 0.0), "lse": lse}
    if op == "loss_grad":
        g = torch.where(given, st["grad_logprob"], 0.0)[:, None]
        d = torch.exp(x.sub_(st["lse"][:, None])).mul_(st["grad_lse"][:, None] - g)
        d.scatter_add_(1, at, g)
        return {"hidden": (d @ w).to(dt), "weight": (d.T @ h).to(dt)}
    if op in NORM_OPS:
        return _plain_norm(st) if op == "norm" else _plain_norm_grad(st)
    q, k, causal = case["queries"], case["keys"], case["causal"]
    bucket = _buckets(case)
    if op == "bias":
        bias = st["table"].float()[bucket].permute(2, 0, 1)
        if causal:
            late = torch.arange(k, device="cuda")[None, :] > torch.arange(k - q, k, device="cuda")[:, None]
            bias = bias.masked_fill(late, -math.inf)
        return bias.to(dt).contiguous()
    grad = st["grad"].float().sum(0)
    if causal:
        late = torch.arange(k, device="cuda")[None, :] > torch.arange(k - q, k, device="cuda")[:, None]
        grad = grad.masked_fill(late, 0.0)
    total = torch.zeros(case["buckets"], case["heads"], device="cuda")
    total.index_add_(0, bucket.reshape(-1), grad.permute(1, 2, 0).reshape(q * k, -1))
    return total.to(dt)


def _buckets(case):
    """The bucket of each pair of query and key, the queries the last ones of the keys.

    Half of the buckets (all, causal) tell distances one by one up to half their
    number; the rest widen in equal ratios up to the largest distance.  The logarithms
    take 64 bits, and a border belongs to the bucket above it."""
    q, k = case["queries"], case["keys"]
    rel = (torch.arange(k, device="cuda")[None, :] - torch.arange(k - q, k, device="cuda")[:, None])
    n = case["buckets"] if case["causal"] else case["buckets"] // 2
    away = (-rel).clamp(min=0) if case["causal"] else rel.abs()
    one = n // 2
    ratio = torch.log(away.clamp(min=1).double() / one) / math.log(case["distance"] / one)
    wide = one + (ratio * (n - one) + 1e-9).floor().long()
    bucket = torch.where(away < one, away, wide.clamp(max=n - 1))
    return bucket if case["causal"] else bucket + n * (rel > 0)


def _f(x):
    return None if x is None else x.float()


def _normed(x, stats, weight, bias):
    """(normalised, with weight and bias)."""
    unit = (x - stats[0]) * stats[1]
    out = unit * weight
    return unit, out if bias is None else out + bias


def _plain_norm(st):
    case, dt = st["case"], DTYPES[st["case"]["dtype"]]
    u = st["block"].float()
    if case["post"]:
        u = _normed(u, _stats(u, case["kind"]), _f(st["block_weight"]), _f(st["block_bias"]))[1]
    if st["gate"] is not None:
        u = u * st["gate"].float()
    x = st["residual"].float() + u * case["scale"]
    y = _normed(x, _stats(x, case["kind"]), _f(st["weight"]), _f(st["bias"]))[1]
    return {"residual": x.to(dt), "out": y.to(dt)}


def _norm_back(g, unit, rstd, weight, kind):
    """The gradient of a norm's input, given that of its output."""
    t = g * weight
    d = t - unit * (t * unit).mean(-1, keepdim=True)
    if kind == "layer":
        d = d - t.mean(-1, keepdim=True)
    return d * rstd


def _plain_norm_grad(st):
    case, dt = st["case"], DTYPES[st["case"]["dtype"]]
    kind, width = case["kind"], case["width"]
    stats = st["stats"].split(1, -1)

    def columns(t):
        return t.reshape(-1, width).sum(0)

    g, block = st["grad_out"].float(), st["block"].float()
    unit, _ = _normed(st["residual"].float(), stats[:2], _f(st["weight"]), None)
    out = {"weight": columns(g * unit)}
    if st["bias"] is not None:
        out["bias"] = columns(g)
    dx = st["grad_residual"].float() + _norm_back(g, unit, stats[1], _f(st["weight"]), kind)
    out["residual"] = dx
    du, u = dx * case["scale"], block
    if case["post"]:
        block_unit, u = _normed(block, stats[2:], _f(st["block_weight"]), _f(st["block_bias"]))
    if st["gate"] is not None:
        dgate = du * u
        out["gate"] = columns(dgate) if st["gate"].dim() == 1 else dgate.sum(1, keepdim=True)
        du = du * st["gate"].float()
    if case["post"]:
        out["block_weight"] = columns(du * block_unit)
        if st["block_bias"] is not None:
            out["block_bias"] = columns(du)
        du = _norm_back(du, block_unit, stats[3], _f(st["block_weight"]), kind)
    out["block"] = du
    return {k: v.to(dt) for k, v in out.items()}


# -- the definition, in 64 bits ---------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op in LOSS_OPS:
        return _exact_loss(case, st)
    if op in NORM_OPS:
        return _exact_norm(case, st)
    q, k = case["queries"], case["keys"]
    # distance by distance: what a query and a key that far apart have in common
    rels = range(-(k - 1), 1 if case["causal"] else q)
    index = torch.tensor([_exact_bucket(case, r) for r in rels], device="cuda")
    rel = torch.arange(k, device="cuda") - torch.arange(k - q, k, device="cuda")[:, None]
    held = rel < len(rels) - (k - 1)
    if op == "bias":
        values = st["table"].double()[index].T.contiguous()
        picked = values[:, (rel + (k - 1)).clamp(max=len(rels) - 1)]
        return torch.where(held, picked, -math.inf)
    total = torch.zeros(case["heads"], len(rels), dtype=torch.float64, device="cuda")
    where = (rel + (k - 1))[held]
    for part in st["grad"]:
        for h in range(case["heads"]):
            total[h].index_add_(0, where, part[h].double()[held])
    table = torch.zeros(case["buckets"], case["heads"], dtype=torch.float64, device="cuda")
    return table.index_add_(0, index, total.T.contiguous())


def _exact_bucket(case, rel):
    """By whole numbers: bucket one + s begins at the least distance a with
    (a / one) ** (n - one) >= (distance / one) ** s."""
    n = case["buckets"] if case["causal"] else case["buckets"] // 2
    start = n if rel > 0 and not case["causal"] else 0
    a, one = abs(rel), n // 2
    if a < one:
        return start + a
    if a >= case["distance"]:
        return start + n - 1
    steps, s = n - one, 0
    while s + 1 < steps and a ** steps * one ** (s + 1) >= case["distance"] ** (s + 1) * one ** steps:
        s += 1
    return start + one + s


def _exact_loss(case, st):
    w = st["weight"].double()
    rows = max(1, (1 << 27) // case["vocab"])
    logprob, lse, dh, dw = [], [], [], torch.zeros_like(w) if case["op"] == "loss_grad" else None
    for at in range(0, case["rows"], rows):
        part = slice(at, at + rows)
        h, t = st["hidden"][part].double(), st["targets"][part]
        logp = torch.log_softmax(torch.mm(h, w.T), 1)
        pick = t.clamp(min=0)[:, None]
        if case["op"] == "loss":
            first = logp[:, :1]
            lse.append((torch.mm(h, w[:1].T) - first)[:, 0])
            logprob.append(torch.where(t == IGNORE, 0.0, logp.gather(1, pick)[:, 0]))
            continue
        g = torch.where(t == IGNORE, 0.0, st["grad_logprob"][part].double())[:, None]
        p = logp.exp_()
        d = p * st["grad_lse"][part].double()[:, None] - p * g
        d.scatter_add_(1, pick, g)
        dh.append(torch.mm(d, w))
        dw.addmm_(d.T, h)
    if case["op"] == "loss":
        return {"logprob": torch.cat(logprob), "lse": torch.cat(lse)}
    return {"hidden": torch.cat(dh), "weight": dw}


def _exact_norm(case, st):
    leaves = {k: st[k].double().requires_grad_(case["op"] == "norm_grad")
              for k in ("residual", "block", "weight", "bias", "block_weight", "block_bias", "gate")
              if st[k] is not None}

    def normed(x, weight, bias):
        if case["kind"] == "layer":
            x = x - x.mean(-1, keepdim=True)
        y = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + EPS) * leaves[weight]
        return y + leaves[bias] if bias in leaves else y

    with torch.set_grad_enabled(case["op"] == "norm_grad"):
        u = leaves["block"]
        if case["post"]:
            u = normed(u, "block_weight", "block_bias")
        u = u * leaves.get("gate", 1.0) * case["scale"]
        if case["op"] == "norm":
            x = leaves["residual"] + u
            return {"residual": x, "out": normed(x, "weight", "bias")}
        # the residual that is at hand already has the block's part
        x = leaves["residual"] + (u - u.detach())
        y = normed(x, "weight", "bias")
        names = list(leaves)
        grads = torch.autograd.grad([x, y], [leaves[k] for k in names],
                                    [st["grad_residual"].double(), st["grad_out"].double()])
    return dict(zip(names, grads))


# -- what a pass cannot do without ------------------------------------------

def work(case):
    op, b = case["op"], BYTES[case["dtype"]]
    if op in LOSS_OPS:
        n, d, v = case["rows"], case["width"], case["vocab"]
        if op == "loss":
            return {"bytes": (n + v) * d * b + 16 * n, "flops": 2 * n * d * v + 4 * n * v}
        return {"bytes": 2 * (n + v) * d * b + 20 * n, "flops": 6 * n * d * v + 4 * n * v}
    if op in NORM_OPS:
        m = case["rows"] * case["width"]
        post = 2 if case["post"] else 0
        layer = 2 if case["kind"] == "layer" else 1
        vectors = (layer * (1 + post // 2) + case["groups"]) * case["width"] * b
        if op == "norm":
            return {"bytes": 4 * m * b + vectors, "flops": (8 + 4 * post) * m}
        return {"bytes": 6 * m * b + 2 * vectors + (2 + post) * 4 * case["rows"],
                "flops": (16 + 8 * post) * m}
    m = case["heads"] * case["queries"] * case["keys"]
    table = case["heads"] * case["buckets"] * b
    if op == "bias":
        return {"bytes": m * b + table, "flops": m}
    return {"bytes": case["batch"] * m * b + table, "flops": case["batch"] * m}
