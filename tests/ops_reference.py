"""Plain 64-bit forms of the language-model operators, written from their
definitions, for the GPU tests to compare with."""

from __future__ import annotations

import math

import torch

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
# half a unit in the last place, relative, and the smallest spacing
HALF_ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


def rounding(value: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """What one rounding of the 64-bit ``value`` to ``dtype`` may be off by."""
    return value.abs() * HALF_ULP[dtype] + TINY[dtype]


def close(got: torch.Tensor, want: torch.Tensor, tol: torch.Tensor, what: str = "") -> None:
    """|got - want| <= tol elementwise; infinities and NaN at the same places."""
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    tol = tol.detach().double().cpu().expand_as(want) if torch.is_tensor(tol) else tol
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    odd = ~fine & ~torch.isnan(want)
    assert torch.equal(got[odd], want[odd]), what
    diff = torch.where(fine, (got - want).abs(), 0.0)
    over = diff > torch.where(fine, tol, 1.0) if torch.is_tensor(tol) else diff > tol
    if bool(over.any()):
        k = int(torch.argmax((diff / tol).reshape(-1) if torch.is_tensor(tol) else diff.reshape(-1)))
        raise AssertionError(
            f"{what}: {int(over.sum())} of {over.numel()} values off; at {k}: got "
            f"{got.reshape(-1)[k].item()!r}, want {want.reshape(-1)[k].item()!r}, difference "
            f"{diff.reshape(-1)[k].item():.3g}")


# -- embedding ---------------------------------------------------------------

def embedding_grad(grad, ids, rows, scale, padding_idx=None):
    """(gradient, sum of magnitudes, tokens per row), 64 bits, on the CPU."""
    width = grad.shape[-1]
    g, t = grad.double().cpu().reshape(-1, width), ids.cpu().reshape(-1).long()
    keep = (t >= 0) & (t < rows)
    if padding_idx is not None:
        keep &= t != padding_idx
    g, t = g[keep], t[keep]
    total = torch.zeros(rows, width, dtype=torch.float64).index_add_(0, t, g)
    size = torch.zeros(rows, width, dtype=torch.float64).index_add_(0, t, g.abs())
    count = torch.bincount(t, minlength=rows)[:, None]
    return total * scale, size * abs(scale), count


# -- log probabilities -------------------------------------------------------

def logprobs(logits, targets, top, ignore_index=-100):
    """{logprob, entropy, lse, top_logprob, top_id} in 64 bits, on the CPU."""
    x = logits.double().cpu().reshape(-1, logits.shape[-1])
    t = targets.cpu().reshape(-1).long()
    n, v = x.shape
    broken = (torch.isnan(x) | (x == math.inf)).any(1)
    most = x.amax(1, keepdim=True)
    empty = ((x == -math.inf).all(1)) & ~broken
    base = torch.where(torch.isfinite(most), most, torch.zeros_like(most))
    total = torch.exp(x - base).sum(1, keepdim=True)
    logp = (x - base) - torch.log(total)
    logp[empty] = -math.inf
    lse = (base + torch.log(total))[:, 0]
    p = torch.exp(logp)
    entropy = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(1)
    good = (t >= 0) & (t < v)
    picked = logp.gather(1, t.clamp(0, v - 1)[:, None])[:, 0]
    picked = torch.where(good, picked, torch.full_like(picked, math.nan))
    for out in (picked, entropy, lse):
        out[broken] = math.nan
    picked[t == ignore_index] = 0.0
    entropy[empty] = 0.0
    lse[empty] = -math.inf
    # NaN above +inf, equal values by rising index
    order = torch.argsort(torch.where(torch.isnan(x), math.inf, x), dim=1, descending=True,
                          stable=True)
    nan_first = torch.argsort(torch.isnan(x).gather(1, order).to(torch.int8), dim=1,
                              descending=True, stable=True)
    top_id = order.gather(1, nan_first)[:, :top]
    top_logprob = logp.gather(1, top_id)
    top_logprob[broken] = math.nan
    shape = tuple(logits.shape[:-1])
    return {"logprob": picked.view(shape), "entropy": entropy.view(shape), "lse": lse.view(shape),
            "top_logprob": top_logprob.view(*shape, top), "top_id": top_id.view(*shape, top)}


def logprobs_grad(logits, targets, grad_logprob, grad_entropy, ignore_index=-100):
    """(gradient, sum of magnitudes of its terms) in 64 bits, on the CPU."""
    x = logits.double().cpu().reshape(-1, logits.shape[-1])
    t = targets.cpu().reshape(-1).long()
    r = logprobs(logits, targets, 0, ignore_index)
    empty = r["lse"].reshape(-1) == -math.inf
    logp = torch.log_softmax(x, 1)
    p = torch.exp(logp)
    g = torch.zeros(len(t), dtype=torch.float64)
    if grad_logprob is not None:
        g = grad_logprob.double().cpu().reshape(-1)
        g = torch.where(t == ignore_index, 0.0, g)
    one = torch.zeros_like(p).scatter_(1, t.clamp(0, x.shape[1] - 1)[:, None], 1.0)
    one[t == ignore_index] = 0.0
    d = g[:, None] * (one - p)
    size = g.abs()[:, None] * (one + p)
    if grad_entropy is not None:
        h = grad_entropy.double().cpu().reshape(-1)[:, None]
        big_h = r["entropy"].reshape(-1)[:, None]
        logp = torch.where(p > 0, logp, torch.zeros_like(logp))
        d = d - h * p * (logp + big_h)
        size = size + h.abs() * p * (logp.abs() + big_h)
    d[empty], size[empty] = 0.0, 0.0
    return d.view(logits.shape), size.view(logits.shape)


# -- 8 bits ------------------------------------------------------------------

def held(x):
    """(codes, exponents, values) of x's 8-bit form, on the CPU; the values in 64 bits."""
    flat = x.detach().double().cpu().reshape(-1)
    n = flat.numel()
    codes, exponents = [], []
    if not n:
        return flat.to(torch.int8), flat.to(torch.uint8), flat
    for block in torch.split(flat, 32):
        if not bool(torch.isfinite(block).all()):
            exponents.append(255)
            codes.append(torch.zeros(len(block), dtype=torch.int8))
            continue
        e = 1
        most = float(block.abs().max())
        if most:
            e = max(1, math.frexp(most)[1] - 1 - 7 + 127)       # one below, then up
            while round(math.ldexp(most, 127 - e)) > 127:
                e += 1
        exponents.append(e)
        codes.append(torch.tensor([round(math.ldexp(float(v), 127 - e)) for v in block],
                                  dtype=torch.int8))
    codes, exponents = torch.cat(codes), torch.tensor(exponents, dtype=torch.uint8)
    return codes, exponents, values(codes, exponents)


def values(codes, exponents):
    e = exponents.cpu().long().repeat_interleave(32)[:codes.numel()]
    step = torch.ldexp(torch.ones(len(e), dtype=torch.float64), e - 127)
    return torch.where(e == 255, math.nan, codes.cpu().double() * step)


def act(x, kind):
    """(f, f', relative error scale of both, sum of magnitudes of f') in 64 bits."""
    x = x.double()
    if kind == "gelu":
        cdf, pdf = 0.5 * torch.special.erfc(-x / math.sqrt(2.0)), torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)
        return x * cdf, cdf + x * pdf, 4 + x * x, cdf + (x * pdf).abs()
    if kind == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        arg = 2 * c * (x + 0.044715 * x ** 3)
        s = torch.sigmoid(arg)
        more = x * s * torch.sigmoid(-arg) * 2 * c * (1 + 3 * 0.044715 * x * x)
        return x * s, s + more, 4 + arg.abs(), s + more.abs()
    s = torch.sigmoid(x)
    return x * s, s + x * s * torch.sigmoid(-x), 4 + x.abs(), s + (x * s * torch.sigmoid(-x)).abs()
