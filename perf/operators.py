"""Timed cases of the language-model operators, ``minispeed_amd.ops``.

Three operators of a training step, each in its directions:

``lookup``, ``lookup_grad``
    the scaled token embedding and the gradient of its table, summed over the
    tokens sorted by id
``logprobs``, ``logprobs_grad``
    the log probability of a given token per row of logits, with the entropy
    and the most likely alternatives, and the gradient of the logits
``pack``, ``act``, ``act_grad``
    activations held in 8 bits (a power-of-two scale for each 32 values)
    between forward and backward: the plain round trip, an activation function
    that leaves its input so with its backward pass after it, and the backward
    pass alone

A case names the operator, its sizes, its element type and what its inputs are
like.  Outputs come whole; what is held in 8 bits shows in the values read
from it and in the gradients.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}
BLOCK = 32                 # values that share a scale
IGNORE = -100
EMBED_OPS = ("lookup", "lookup_grad")
LOGIT_OPS = ("logprobs", "logprobs_grad")
ACT_OPS = ("pack", "act", "act_grad")


def listed():
    return [
        # one micro-batch of the tiny GPT (vocab 512, width 256, 8 x 128
        # tokens): the table and the output stay in the caches
        dict(name="lookup-tiny", op="lookup", tokens=1024, width=256, vocab=512, dtype="fp32",
             scaled=False, pad=0.0),
        # 4 x 2048 tokens into the 1.3B GPT
        dict(name="lookup-1.3b", op="lookup", tokens=8192, width=2048, vocab=50257, dtype="fp16",
             scaled=True, pad=0.0),
        # the tiny GPT's backward: launches and the sort count
        dict(name="lookup-grad-tiny", op="lookup_grad", tokens=1024, width=256, vocab=512,
             dtype="fp32", scaled=False, pad=0.0),
        # 16 x 1024 tokens of the 124M GPT, a third of them padding that all
        # falls on one row of the table
        dict(name="lookup-grad-124m", op="lookup_grad", tokens=16384, width=768, vocab=50257,
             dtype="bf16", scaled=True, pad=0.33),
        # 8192 tokens of the 8B decoder: nearly all of the table's gradient is zeros
        dict(name="lookup-grad-8b", op="lookup_grad", tokens=8192, width=4096, vocab=128256,
             dtype="bf16", scaled=False, pad=0.0),
        # sampling: the next token of four sequences with 20 alternatives
        dict(name="logprobs-few", op="logprobs", rows=4, vocab=50257, dtype="bf16", top=20,
             entropy=True, masked=0.0, ignored=0.0),
        # the loss of 8 x 1024 tokens of the 124M GPT, prompts left out of it
        dict(name="logprobs-124m", op="logprobs", rows=8192, vocab=50257, dtype="fp16", top=0,
             entropy=False, masked=0.0, ignored=0.1),
        # scoring 2048 tokens over the 8B decoder's vocabulary with entropy and
        # 8 alternatives, under a vocabulary mask that leaves one row nothing
        dict(name="logprobs-8b", op="logprobs", rows=2048, vocab=128256, dtype="bf16", top=8,
             entropy=True, masked=0.3, ignored=0.0),
        # the backward pass of the 124M loss with an entropy bonus
        dict(name="logprobs-grad-124m", op="logprobs_grad", rows=8192, vocab=50257, dtype="fp16",
             top=0, entropy=True, masked=0.0, ignored=0.1),
        # the tiny GPT's MLP (1024 tokens, 4 x 256 wide), backward
        dict(name="act-grad-tiny", op="act_grad", rows=1024, width=1024, dtype="fp32", kind="gelu"),
        # the 1.3B GPT's MLP: 8192 tokens, 4 x 2048 wide, forward and backward
        dict(name="act-1.3b", op="act", rows=8192, width=8192, dtype="fp16", kind="gelu"),
        # the 8B decoder's gated MLP: 4096 tokens, 14336 wide, backward
        dict(name="act-grad-8b", op="act_grad", rows=4096, width=14336, dtype="bf16", kind="swiglu"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(EMBED_OPS + LOGIT_OPS + ACT_OPS)
    dtype = rng.choice(("fp32", "fp16", "bf16"))
    if op in EMBED_OPS:
        width = _log_int(rng, 64, 4096)
        if rng.random() < 0.75:                    # most widths are whole vectors
            width = max(64, width // 64 * 64)
        vocab = _log_int(rng, 512, 128256)
        while vocab * width * BYTES[dtype] > 1.06e9:
            vocab //= 2
        tokens = _log_int(rng, 1, 16384)
        return dict(op=op, tokens=tokens, width=width, vocab=vocab, dtype=dtype,
                    scaled=rng.random() < 0.5, pad=rng.choice((0.0, 0.0, 0.33, 0.9)))
    if op in LOGIT_OPS:
        vocab = _log_int(rng, 512, 128256)
        rows = _log_int(rng, 1, 8192)
        while rows * vocab * BYTES[dtype] > 8.2e8:
            rows = max(1, rows // 2)
        top = rng.choice((0, 1, 5, 20, 50)) if op == "logprobs" else 0
        return dict(op=op, rows=rows, vocab=vocab, dtype=dtype, top=top,
                    entropy=rng.random() < 0.5, masked=rng.choice((0.0, 0.0, 0.3)),
                    ignored=rng.choice((0.0, 0.1)))
    width = _log_int(rng, 256, 14336)
    if rng.random() < 0.75:
        width = width // 64 * 64
    rows = _log_int(rng, 1, 8192)
    while rows * width * BYTES[dtype] > 1.2e8:
        rows = max(1, rows // 2)
    case = dict(op=op, rows=rows, width=width, dtype=dtype, kind="none")
    if op != "pack":
        case["kind"] = rng.choice(("gelu", "gelu_tanh", "silu", "swiglu"))
    return case


# -- inputs -----------------------------------------------------------------

def _zipf(vocab):
    p = 1.0 / (np.arange(vocab) + 2.7)
    return p / p.sum()


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def prepare(case, seed):
    g = _gen(seed)
    dt, op = DTYPES[case["dtype"]], case["op"]

    def randn(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(std).to(dt)

    if op in EMBED_OPS:
        n, d, v = case["tokens"], case["width"], case["vocab"]
        # token frequencies as in text, the frequent ids anywhere in the table
        cdf = torch.from_numpy(np.cumsum(_zipf(v))).to("cuda")
        u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
        rank = torch.searchsorted(cdf, u).clamp_(max=v - 1)
        ids = torch.randperm(v, generator=g, device="cuda")[rank]
        if case["pad"]:
            padded = torch.rand(n, generator=g, device="cuda") < case["pad"]
            ids = torch.where(padded, torch.full_like(ids, v // 2), ids)
        st = {"case": case, "ids": ids, "rows": v, "scale": math.sqrt(d) if case["scaled"] else 1.0}
        if op == "lookup":
            st["weight"] = randn(v, d, std=0.02)
        else:
            st["grad"] = randn(n, d, std=1e-2)
        return st

    if op in LOGIT_OPS:
        n, v = case["rows"], case["vocab"]
        logits = torch.randn(n, v, generator=g, device="cuda", dtype=dt)
        logits.mul_(2.5)
        targets = torch.randint(0, v, (n,), generator=g, device="cuda")
        # the given token is likely, as in a trained model
        logits.scatter_add_(1, targets[:, None], torch.full((n, 1), 6.0, dtype=dt, device="cuda"))
        if case["masked"]:
            gone = torch.rand(v, generator=g, device="cuda") < case["masked"]
            logits.masked_fill_(gone, -math.inf)
            if n > 3:
                logits[n // 2] = -math.inf          # a row whose mask leaves nothing
        if case["ignored"]:
            out = torch.rand(n, generator=g, device="cuda") < case["ignored"]
            targets = torch.where(out, torch.full_like(targets, IGNORE), targets)
        st = {"case": case, "logits": logits, "targets": targets}
        if op == "logprobs_grad":
            # what the forward pass left, and the gradients that come down
            f = logits.float()
            st["lse"] = torch.logsumexp(f, 1)
            st["grad_logprob"] = torch.randn(n, generator=g, device="cuda") * 0.1 - 1.0
            if case["entropy"]:
                logp = f.sub_(st["lse"][:, None])
                st["entropy"] = -(logp.exp() * logp).nan_to_num_(0.0).sum(1)
                st["grad_entropy"] = torch.randn(n, generator=g, device="cuda") * 0.01
        return st

    n, w = case["rows"], case["width"]
    # pre-activations: each channel has a spread of its own, some far larger
    spread = torch.exp(torch.randn(w, generator=g, device="cuda") * 0.7)

    def hidden():
        h = torch.randn(n, w, generator=g, device="cuda") * spread
        return h.to(dt)

    st = {"case": case, "h": hidden()}
    if case["kind"] == "swiglu":
        st["up"] = hidden()
    if op != "pack":
        st["grad"] = randn(n, w, std=1e-2)
    if op == "act_grad":
        # what the forward pass holds: whole numbers of 8 bits, and the byte of
        # the exponent of each block's scale
        st["saved"] = [_codes(st[k]) for k in ("h", "up") if k in st]
        for k in ("h", "up"):
            st.pop(k, None)
        st["shape"] = (n, w)
    return st


def _codes(x):
    """The 8-bit form of x: (codes [n] int8, exponents [blocks] uint8)."""
    flat = x.reshape(-1).float()
    n = flat.numel()
    flat = torch.nn.functional.pad(flat, (0, -n % BLOCK)).view(-1, BLOCK)
    bits = flat.abs().amax(1).view(torch.int32)
    exp = ((bits + 0x10000 >> 23) - 6).clamp_(min=1)
    exp = torch.where(bits >= 0x7F800000, torch.full_like(exp, 255), exp)
    step = (254 - exp.clamp(max=253) << 23).view(torch.float32)      # 2 ** (127 - exp)
    codes = (flat * step[:, None]).round_().masked_fill_((exp == 255)[:, None], 0.0)
    return codes.to(torch.int8).view(-1)[:n].contiguous(), exp.to(torch.uint8)


def _values(codes, exp):
    """The values that codes stand for, in 32 bits."""
    n = codes.numel()
    e = exp.to(torch.int32)
    step = (e << 23).view(torch.float32)
    step = torch.where(e == 255, torch.full_like(step, math.nan), step)
    c = torch.nn.functional.pad(codes, (0, -n % BLOCK)).view(-1, BLOCK).float()
    return (c * step[:, None]).view(-1)[:n]


# -- one pass ---------------------------------------------------------------

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(st):
    import minispeed_amd as ms
    ops, case = ms.ops, st["case"]
    op = case["op"]
    if op == "lookup":
        return ops.embedding(st["ids"], st["weight"], scale=st["scale"])
    if op == "lookup_grad":
        return ops.embedding_grad(st["grad"], st["ids"], st["rows"], scale=st["scale"])
    if op == "logprobs":
        r = ops.token_logprobs(st["logits"], st["targets"], top=case["top"],
                               entropy=case["entropy"], ignore_index=IGNORE)
        out = {"logprob": r.logprob, "lse": r.lse}
        if case["entropy"]:
            out["entropy"] = r.entropy
        if case["top"]:
            out["top_logprob"], out["top_id"] = r.top_logprob, r.top_id
        return out
    if op == "logprobs_grad":
        return ops.token_logprobs_grad(st["logits"], st["targets"], st["lse"], st["grad_logprob"],
                                       entropy=st.get("entropy"),
                                       grad_entropy=st.get("grad_entropy"), ignore_index=IGNORE)
    if op == "pack":
        return ops.unpack8(ops.pack8(st["h"]))
    if op == "act":
        first, saved = ops.activation8(st["h"], case["kind"], up=st.get("up"))
        grads, again = ops.activation8_grad(saved, st["grad"], case["kind"])
        return {"first": first, "grads": list(grads), "a": again}
    saved = tuple(ops.Checkpoint8(c, e, st["shape"], st["grad"].dtype) for c, e in st["saved"])
    grads, again = ops.activation8_grad(saved, st["grad"], case["kind"])
    return {"grads": list(grads), "a": again}


def _run_plain(st):
    case = st["case"]
    op, dt = case["op"], DTYPES[case["dtype"]]
    if op == "lookup":
        return (st["weight"][st["ids"]].float() * st["scale"]).to(dt)
    if op == "lookup_grad":
        g = st["grad"].float()
        total = torch.zeros(st["rows"], g.shape[1], device="cuda")
        total.index_add_(0, st["ids"], g)
        return (total * st["scale"]).to(dt)
    if op in LOGIT_OPS:
        x, targets = st["logits"].float(), st["targets"]
        given = targets != IGNORE
        at = targets.clamp(min=0)[:, None]
    if op == "logprobs":
        most = x.amax(1, keepdim=True)
        empty = most == -math.inf
        most = most.masked_fill(empty, 0.0)
        e = torch.exp(x - most)
        total = e.sum(1, keepdim=True)
        lse = (most + torch.log(total))[:, 0]
        picked = x.gather(1, at)[:, 0]
        logp = torch.where(empty[:, 0], picked, picked - lse)
        out = {"logprob": torch.where(given, logp, 0.0), "lse": lse}
        if case["entropy"]:
            mean = (e * (x - most).masked_fill(e == 0, 0.0)).sum(1, keepdim=True) / total
            out["entropy"] = (torch.log(total) - mean).masked_fill(empty, 0.0)[:, 0]
        if case["top"]:
            value, index = torch.sort(x, dim=1, descending=True, stable=True)
            value, index = value[:, :case["top"]], index[:, :case["top"]]
            out["top_logprob"] = torch.where(empty, value, value - lse[:, None])
            out["top_id"] = index.contiguous()
        return out
    if op == "logprobs_grad":
        lse = st["lse"]
        empty = lse == -math.inf
        logp = x - lse.masked_fill(empty, 0.0)[:, None]
        p = torch.exp(logp)
        g = torch.where(given, st["grad_logprob"], 0.0).masked_fill(empty, 0.0)
        d = -p * g[:, None]
        d.scatter_add_(1, at, g[:, None])
        if case["entropy"]:
            h, gh = st["entropy"][:, None], st["grad_entropy"][:, None]
            d = d - gh * p * (logp.masked_fill(p == 0, 0.0) + h)
        return d.to(dt)
    if op == "pack":
        return _values(*_codes(st["h"])).view(st["h"].shape).to(dt)
    if op == "act":
        first = _act(st["h"].float(), case["kind"])[0]
        saved = [_codes(st["h"])]
        if case["kind"] == "swiglu":
            first = first * st["up"].float()
            saved.append(_codes(st["up"]))
        return {"first": first.to(dt), **_plain_act_grad(case, saved, st["grad"])}
    return _plain_act_grad(case, st["saved"], st["grad"])


def _plain_act_grad(case, saved, grad):
    h = _values(*saved[0]).view(grad.shape)
    f, df = _act(h, case["kind"])
    g, dt = grad.float(), grad.dtype
    if case["kind"] != "swiglu":
        return {"grads": [(g * df).to(dt)], "a": f.to(dt)}
    u = _values(*saved[1]).view(grad.shape)
    return {"grads": [(g * u * df).to(dt), (g * f).to(dt)], "a": (f * u).to(dt)}


def _act(x, kind):
    """The activation and its derivative, elementwise."""
    if kind == "gelu":
        cdf = 0.5 * torch.erfc(x * -math.sqrt(0.5))
        return x * cdf, cdf + x * torch.exp(-0.5 * x * x) * (1.0 / math.sqrt(2.0 * math.pi))
    if kind == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        s = 1.0 / (1.0 + torch.exp(-2.0 * c * (x + 0.044715 * x * x * x)))
        return x * s, s + x * s * (1.0 - s) * 2.0 * c * (1.0 + 3.0 * 0.044715 * x * x)
    s = 1.0 / (1.0 + torch.exp(-x))
    return x * s, s * (1.0 + x * (1.0 - s))


# -- the definition, in 64 bits ---------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    op, f64 = case["op"], torch.float64
    if op == "lookup":
        return torch.index_select(st["weight"].to(f64), 0, st["ids"]) * st["scale"]
    if op == "lookup_grad":
        total = torch.zeros(st["rows"], case["width"], dtype=f64, device="cuda")
        order = torch.argsort(st["ids"], stable=True)
        total.index_add_(0, st["ids"][order], st["grad"][order].to(f64))
        return total.mul_(st["scale"])
    if op == "logprobs":
        parts = [_exact_logprobs(case, x, t) for x, t in _pieces(st["logits"], st["targets"])]
        return {k: None if parts[0][k] is None else torch.cat([p[k] for p in parts])
                for k in parts[0]}
    if op == "logprobs_grad":
        out, at = [], 0
        for x, t in _pieces(st["logits"], st["targets"]):
            s = slice(at, at + x.shape[0])
            at += x.shape[0]
            h = (st["entropy"][s], st["grad_entropy"][s]) if case["entropy"] else None
            out.append(_exact_grad(x.to(f64), t, st["grad_logprob"][s], h))
        return torch.cat(out)
    if op == "pack":
        return _exact_held(st["h"]).view(st["h"].shape)
    out = {}
    if op == "act":
        out["first"] = _exact_act(st["h"].to(f64), case["kind"])
        if case["kind"] == "swiglu":
            out["first"] *= st["up"].to(f64)
        values = [_exact_held(st[k]).view(st["h"].shape) for k in ("h", "up") if k in st]
    else:
        values = [(c.to(f64) * _pow2(e.to(torch.int64) - 127).repeat_interleave(BLOCK)[:c.numel()])
                  .view(st["shape"]) for c, e in st["saved"]]
    with torch.enable_grad():
        values = [x.requires_grad_() for x in values]
        a = _exact_act(values[0], case["kind"])
        if case["kind"] == "swiglu":
            a = a * values[1]
        grads = torch.autograd.grad(a, values, st["grad"].to(f64))
    return {**out, "grads": list(grads), "a": a.detach()}


def _pow2(e):
    """2 ** e in 64 bits, for whole e of any sign."""
    return (e.to(torch.int64) + 1023 << 52).view(torch.float64)


def _pieces(logits, targets):
    rows = max(1, (1 << 26) // logits.shape[1])
    for at in range(0, logits.shape[0], rows):
        yield logits[at:at + rows], targets[at:at + rows]


def _exact_logprobs(case, x, t):
    x = x.to(torch.float64)
    lse = torch.logsumexp(x, 1)
    logp = torch.where(lse[:, None] == -math.inf, x, x - lse[:, None])
    picked = logp.gather(1, t.clamp(min=0)[:, None])[:, 0]
    out = {"logprob": torch.where(t == IGNORE, 0.0, picked), "lse": lse}
    if case["entropy"]:
        out["entropy"] = torch.special.entr(torch.exp(logp)).sum(1)
    if case["top"]:
        out["top_logprob"] = torch.topk(logp, case["top"], dim=1).values
        out["top_id"] = None
    return out


def _exact_grad(x, t, g, entropy):
    p = torch.softmax(x, 1).nan_to_num(0.0)
    one = torch.zeros_like(p).scatter_(1, t.clamp(min=0)[:, None], 1.0)
    alive = p.sum(1, keepdim=True) > 0
    g = torch.where(t == IGNORE, 0.0, g.to(torch.float64))[:, None]
    d = torch.where(alive, g * (one - p), 0.0)
    if entropy is not None:
        h = torch.special.entr(p).sum(1, keepdim=True)
        d += entropy[1].to(torch.float64)[:, None] * (torch.special.entr(p) - p * h)
    return d


def _exact_held(x):
    x = x.reshape(-1).to(torch.float64)
    n = x.numel()
    x = torch.cat([x, x.new_zeros(-n % BLOCK)]).view(-1, BLOCK)
    most = x.abs().amax(1, keepdim=True)
    exponent = torch.frexp(most).exponent - 7                  # most in [64, 128) steps
    exponent += torch.round(most * _pow2(-exponent)) > 127
    exponent = exponent.clamp(min=-126)
    return (torch.round(x * _pow2(-exponent)) * _pow2(exponent)).view(-1)[:n]


def _exact_act(x, kind):
    if kind == "gelu":
        return x * torch.special.ndtr(x)
    if kind == "gelu_tanh":
        return 0.5 * x * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (x + 0.044715 * x ** 3)))
    return x * torch.sigmoid(x)


# -- what a pass cannot do without ------------------------------------------

def _distinct(case):
    """The expected number of different ids among the case's tokens."""
    p = (1.0 - case["pad"]) * _zipf(case["vocab"])
    seen = float(-np.expm1(case["tokens"] * np.log1p(-p)).sum())
    return min(case["tokens"], case["vocab"], seen + (1.0 if case["pad"] else 0.0))


def work(case):
    op, b = case["op"], BYTES[case["dtype"]]
    if op in EMBED_OPS:
        n, d = case["tokens"], case["width"]
        ids = 8 * n
        if op == "lookup":
            return {"bytes": ids + (_distinct(case) + n) * d * b, "flops": n * d}
        return {"bytes": ids + (n + case["vocab"]) * d * b, "flops": n * d}
    if op in LOGIT_OPS:
        n, v = case["rows"], case["vocab"]
        if op == "logprobs":
            row = 16 + 4 * case["entropy"] + 12 * case["top"]
            return {"bytes": n * v * b + n * row, "flops": (4 + 2 * case["entropy"]) * n * v}
        return {"bytes": 2 * n * v * b + n * (16 + 8 * case["entropy"]),
                "flops": (4 + 2 * case["entropy"]) * n * v}
    m = case["rows"] * case["width"]
    held = m + -(-m // BLOCK)
    both = 2 if case["kind"] == "swiglu" else 1
    if op == "pack":
        return {"bytes": 2 * m * b + 2 * held, "flops": 4 * m}
    if op == "act":      # the 8-bit form is written by one pass and read by the other
        return {"bytes": (2 * both + 3) * m * b + 2 * both * held, "flops": 40 * both * m}
    return {"bytes": (both + 2) * m * b + both * held, "flops": 24 * both * m}
