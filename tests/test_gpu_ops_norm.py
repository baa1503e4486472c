"""Norms around a block, and their gradients, against autograd in 64 bits.

Tolerances, u = 2^-24.  Statistics of W values: W u / 2 of the mean of magnitudes and of
squares (sums in 32 bits), so a normalised value v is off by (W / 2 + 8) u (|v| + mean / deviation
+ 1).  Results add a few u of the magnitudes that meet, and one rounding.  Gradients: the same
for each of the terms that meet in a value; sums over R rows (R + 8) u of the sum of
magnitudes more.  Sums here are made in some dozens of partial sums, so W / 2 and R are
far on the safe side, and beside them the statistics from the forward pass, of the
residual before it is rounded, are off by half an ulp of the type over sqrt(W) and more:
half an ulp of each term is allowed for that.
"""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import minispeed_amd as ms
from minispeed_amd import build
from tests import ops_reference as ref
from tests.test_ops_abi import Rows

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
NAMES = ("residual", "block", "weight", "bias", "block_weight", "block_bias", "gate")


def make(shape, dtype, seed, kind="layer", post=True, gate=None, block=True, bias=True):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt, w = ref.DTYPES[dtype], shape[-1]

    def randn(*size, std=1.0, mean=0.0):
        return (torch.randn(*size, generator=g, device=DEV) * std + mean).to(dt)

    spread = torch.exp(torch.randn(w, generator=g, device=DEV) * 0.7)
    layer = kind == "layer" and bias
    return {"residual": (randn(*shape).float() * spread + 0.2).to(dt),
            "block": randn(*shape, std=0.7) if block else None,
            "weight": randn(w, std=0.2, mean=1.0), "bias": randn(w, std=0.2) if layer else None,
            "block_weight": randn(w, std=0.2, mean=1.0) if post else None,
            "block_bias": randn(w, std=0.2) if post and layer else None,
            "gate": None if gate is None else randn(*gate, std=0.3, mean=0.5)}


def formula(o, scale, eps, kind):
    """(next, out, normalised values) in 64 bits, of the double tensors in o."""
    def normed(x, weight, bias):
        if kind == "layer":
            x = x - x.mean(-1, keepdim=True)
        v = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
        y = v * weight
        return v, y if bias is None else y + bias

    x = o["residual"]
    if o["block"] is not None:
        u = o["block"]
        if o["block_weight"] is not None:
            u = normed(u, o["block_weight"], o["block_bias"])[1]
        if o["gate"] is not None:
            u = u * o["gate"]
        x = x + scale * u
    v, y = normed(x, o["weight"], o["bias"])
    return x, y, v


def doubles(o, grad=False):
    return {k: None if t is None else t.detach().double().requires_grad_(grad) for k, t in o.items()}


def off(x):
    """How much a row's normalised values move, in units of u, per unit of |v| + 1."""
    w = x.shape[-1]
    sd = x.std(-1, unbiased=False, keepdim=True) if w > 1 else x.abs()
    lean = x.mean(-1, keepdim=True).abs() / sd.clamp(min=1e-3)
    return (w / 2 + 8) * (1 + lean)


def call(o, scale, eps, kind):
    if o["block"] is None:
        return None, ms.ops.norm(o["residual"], o["weight"], o["bias"], eps=eps, kind=kind)
    r = ms.ops.residual_norm(o["residual"], o["block"], o["weight"], bias=o["bias"],
                             block_weight=o["block_weight"], block_bias=o["block_bias"], gate=o["gate"],
                             scale=scale, eps=eps, kind=kind)
    return r.residual, r.out


def check(o, kind, scale=0.75, eps=1e-5, only=None, seed=0):
    dt = o["residual"].dtype
    d = doubles(o, True)
    x, y, v = formula(d, scale, eps, kind)
    leaves = {k: None if t is None else t.detach().clone(memory_format=torch.preserve_format).requires_grad_()
              for k, t in o.items()}
    nxt, out = call(leaves, scale, eps, kind)
    move = 1.0
    if o["block"] is not None:
        size = d["block"].abs() if o["block_weight"] is None else \
            (x - d["residual"]).abs() + scale * 2
        t = 16 * U * (x.abs() + size) + ref.rounding(x, dt)
        if o["block_weight"] is not None:
            factor = d["block_weight"].abs() * (d["gate"].abs() if o["gate"] is not None else 1.0) * abs(scale)
            t = t + off(d["block"]) * U * 8 * factor
        ref.close(nxt, x, t, "next")
        if o["block_weight"] is not None:
            move = 1 + off(d["block"]) * 4
    wide = (v.abs() + 1) * d["weight"].abs() + (0 if o["bias"] is None else d["bias"].abs())
    ref.close(out, y, U * (off(x) + 16 + move) * wide + ref.rounding(y, dt), "out")

    g = torch.Generator(device=DEV).manual_seed(seed + 99)
    gy = torch.randn(out.shape, generator=g, device=DEV).to(dt)
    gx = torch.randn(out.shape, generator=g, device=DEV).to(dt)
    ends = [(out, y, gy)] if nxt is None else [(nxt, x, gx), (out, y, gy)]
    if only is not None:
        ends = [ends[only]]
    torch.autograd.backward([a for a, _, _ in ends], [c for _, _, c in ends])
    names = [k for k in NAMES if d[k] is not None]
    want = torch.autograd.grad([b for _, b, _ in ends], [d[k] for k in names],
                               [c.double() for _, _, c in ends], allow_unused=True)
    # sizes of the terms, by the formula with magnitudes in the place of values
    rows = out.numel() // out.shape[-1]
    if kind == "rms":
        rstd = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    else:
        rstd = 1 / torch.sqrt(x.var(-1, unbiased=False, keepdim=True) + eps)
    # Backward has the new residual as it was rounded, x (1 + r) with |r| <= half an ulp, and
    # the statistics of x: its v = (x (1 + r) - mean) rstd is off by |x| rstd half ulps.
    vv = v.abs() + 1 + x.abs() * rstd
    t1 = (gy.double().abs() * d["weight"].abs()) if only in (None, 1) or nxt is None else torch.zeros_like(y)
    along = t1 + vv * (t1 * vv).mean(-1, keepdim=True) + t1.mean(-1, keepdim=True)
    dx = along * rstd + (gx.double().abs() if nxt is not None and only in (None, 0) else 0)
    half = ref.HALF_ULP[dt] * 4 + U * (off(x).amax() + move.amax() if torch.is_tensor(move) else off(x).amax()) * 4
    sizes = {"residual": dx}
    over = lambda q: q.reshape(-1, q.shape[-1]).sum(0) * (1 + rows * U / half)  # noqa: E731
    sizes["weight"] = over(gy.double().abs() * vv)
    sizes["bias"] = over(gy.double().abs())
    if o["block"] is not None:
        q = dx * abs(scale)
        b = d["block"]
        u = b.abs()
        if o["block_weight"] is not None:
            bm = b - b.mean(-1, keepdim=True) if kind == "layer" else b
            br = 1 / torch.sqrt((bm * bm).mean(-1, keepdim=True) + eps)
            bv = (bm * br).abs() + 1
            u = bv * d["block_weight"].abs() + (d["block_bias"].abs() if o["block_bias"] is not None else 0)
        if o["gate"] is not None:
            full = (q * u).expand(out.shape)
            lead = [k for k in range(out.dim() - 1) if o["gate"].dim() == 1 or o["gate"].shape[k] == 1]
            sizes["gate"] = (full.sum(lead, keepdim=o["gate"].dim() > 1) if lead else full) * (1 + rows * U / half)
            q = q * d["gate"].abs()
        if o["block_weight"] is not None:
            sizes["block_weight"], sizes["block_bias"] = over(q * bv), over(q)
            q = q * d["block_weight"].abs()
            q = (q + bv * (q * bv).mean(-1, keepdim=True) + q.mean(-1, keepdim=True)) * br
        sizes["block"] = q
    for name, w in zip(names, want):
        got = leaves[name].grad
        if w is None:
            w = torch.zeros_like(d[name])
        assert got.shape == o[name].shape and got.dtype == dt
        ref.close(got, w, sizes[name].expand(w.shape) * half + ref.rounding(w, dt), f"d{name} {kind}")
    return [t for t in (nxt, out) if t is not None] + [leaves[k].grad for k in names]


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("rows,width", [(1, 64), (3, 1), (5, 7), (70, 256), (33, 257), (17, 1000), (9, 1024),
                                        (40, 2048), (6, 2056), (5, 4096), (3, 5001), (4, 8192)])
def test_sizes(dtype, kind, post, rows, width):
    check(make((rows, width), dtype, rows + width, kind, post), kind)


@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
@pytest.mark.parametrize("kind,post", [("rms", False), ("layer", True)])
def test_the_widest_rows(dtype, kind, post):
    check(make((3, 16384), dtype, 1, kind, post, gate=(16384,)), kind)
    check(make((2, 12289), dtype, 2, kind, post), kind)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("shape,gate", [((6, 40, 96), (96,)), ((6, 40, 96), (6, 1, 96)),
                                        ((6, 40, 96), (6, 40, 96)), ((6, 40, 96), (1, 1, 96)),
                                        ((300, 3, 64), (300, 1, 64)), ((2, 900, 520), (2, 1, 520)),
                                        ((2, 3, 4, 64), (2, 3, 1, 64)), ((5000, 64), (64,)),
                                        ((7, 701, 1100), (7, 1, 1100)), ((1, 1, 2100), (1, 1, 2100))])
def test_gates(dtype, post, shape, gate):
    check(make(shape, dtype, sum(shape), "layer", post, gate), "layer")


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_the_norm_alone(dtype):
    for kind in ("rms", "layer"):
        for shape in ((4, 33), (3, 5, 768), (2000, 128)):
            check(make(shape, dtype, 3, kind, False, block=False), kind)
    check(make((9, 64), dtype, 4, "layer", False, block=False, bias=False), "layer")


def test_one_result_alone_has_a_gradient():
    for only in (0, 1):
        for post in (False, True):
            check(make((30, 200), "fp32", 5, "layer", post, (200,)), "layer", only=only)


def test_layouts():
    o = make((6, 10, 72), "bf16", 6, gate=(6, 1, 72))
    first = check(o, "layer")
    base = torch.zeros(6, 10, 75, dtype=torch.bfloat16, device=DEV)
    for name in ("residual", "block"):
        p = dict(o)
        p[name] = base.clone()[:, :, 2:74]
        p[name].copy_(o[name])
        assert all(torch.equal(a, b) for a, b in zip(check(p, "layer"), first))
        p[name] = o[name].transpose(0, 1).contiguous().transpose(0, 1)
        assert all(torch.equal(a, b) for a, b in zip(check(p, "layer"), first))
    p = dict(o)
    p["weight"] = torch.stack([o["weight"]] * 2, 1)[:, 0]
    p["gate"] = torch.cat([o["gate"]] * 2, 2)[:, :, 72:]
    assert all(torch.equal(a, b) for a, b in zip(check(p, "layer"), first))
    # gradients that come down expanded or strided
    a = {k: t.clone().requires_grad_() for k, t in o.items()}
    r = ms.ops.residual_norm(a["residual"], a["block"], a["weight"], a["bias"], a["block_weight"],
                             a["block_bias"], a["gate"], kind="layer")
    r.out.sum().backward()
    g = ms.ops.residual_norm_grad(torch.ones_like(r.out), None, r.residual.detach(), r.stats,
                                  *(o[k] for k in NAMES[1:]), kind="layer")
    for k in NAMES:
        assert torch.equal(a[k].grad, getattr(g, k)), k


def test_no_rows():
    o = make((0, 64), "fp32", 7, gate=(64,))
    leaves = {k: t.requires_grad_() for k, t in o.items()}
    nxt, out = call(leaves, 1.0, 1e-5, "layer")
    assert nxt.shape == out.shape == (0, 64)
    (nxt.sum() + out.sum()).backward()
    for k in ("weight", "bias", "block_weight", "block_bias", "gate"):
        assert torch.equal(leaves[k].grad, torch.zeros(64, device=DEV)), k
    o = make((0, 5, 64), "bf16", 8, gate=(0, 1, 64))
    leaves = {k: t.requires_grad_() for k, t in o.items()}
    nxt, out = call(leaves, 1.0, 1e-5, "layer")
    out.sum().backward()
    assert leaves["gate"].grad.shape == (0, 1, 64) and not leaves["weight"].grad.any()


def test_large_means_lose_nothing():
    """Rows far from zero: the variance is of the differences from the mean."""
    o = make((20, 512), "fp32", 9, "layer", False, block=False)
    o["residual"] = o["residual"] + 4096.0
    check(o, "layer")


def test_constant_and_zero_rows():
    for dtype in ("fp32", "fp16"):
        o = make((4, 96), dtype, 10, "layer", True)
        o["residual"][0], o["block"][0] = 0.0, 0.0
        o["residual"][1], o["block"][1] = 2.0, 3.0
        nxt, out = call(o, 1.0, 1e-5, "layer")
        _, want, _ = formula(doubles(o), 1.0, 1e-5, "layer")
        assert torch.isfinite(out).all()
        # (a constant block has the norm 0 exactly in 64 bits; in 32 its mean is off by 96 u of 3)
        assert float((out[0].double() - want[0]).abs().max()) < 1e-2
        g = ms.ops.residual_norm_grad(torch.ones_like(out), None, nxt,
                                      ms.ops.residual_norm(**{k: v for k, v in o.items() if v is not None},
                                                           kind="layer").stats,
                                      o["block"], o["weight"], o["bias"], o["block_weight"],
                                      o["block_bias"], kind="layer")
        assert torch.isfinite(g.residual).all() and torch.isfinite(g.block).all()


def test_nan_and_infinity_stay_in_their_rows():
    o = make((40, 300), "fp32", 11, "layer", True, (300,))
    good = call(o, 1.0, 1e-5, "layer")
    o["residual"][3, 5], o["block"][9, 299] = math.nan, math.inf
    nxt, out = call(o, 1.0, 1e-5, "layer")
    keep = torch.ones(40, dtype=torch.bool, device=DEV)
    keep[3] = keep[9] = False
    assert torch.equal(out[keep], good[1][keep]) and torch.equal(nxt[keep], good[0][keep])
    assert out[3].isnan().all() and out[9].isnan().all()


def test_the_same_bits_every_time_and_on_another_stream():
    o = make((700, 6, 520), "fp16", 12, gate=(700, 1, 520))
    r = ms.ops.residual_norm(**o, kind="layer")
    g = torch.randn(700, 6, 520, device=DEV).half()
    rest = [o[k] for k in NAMES[1:]]
    first = ms.ops.residual_norm_grad(g, g, r.residual, r.stats, *rest, kind="layer")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(side):
            again = ms.ops.residual_norm(**o, kind="layer")
            more = ms.ops.residual_norm_grad(g, g, again.residual, again.stats, *rest, kind="layer")
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((*r, *first), (*again, *more)))


def test_differences():
    """The gradients against central differences of the formula in 64 bits."""
    o = make((4, 3, 24), "fp32", 13, gate=(4, 1, 24))
    leaves = {k: t.clone().requires_grad_() for k, t in o.items()}
    r = ms.ops.residual_norm(**leaves, scale=0.6, kind="layer")
    g = torch.Generator(device=DEV).manual_seed(14)
    a, b = (torch.randn(4, 3, 24, generator=g, device=DEV) for _ in range(2))
    ((r.residual * a).sum() + (r.out * b).sum()).backward()

    def loss(z):
        x, y, _ = formula(z, 0.6, 1e-5, "layer")
        return float((x * a).sum() + (y * b).sum())

    step = 1e-5
    for name in NAMES:
        v = torch.randn(o[name].shape, generator=g, device=DEV).double()
        up, down = doubles(o), doubles(o)
        up[name], down[name] = up[name] + step * v, down[name] - step * v
        slope = (loss(up) - loss(down)) / (2 * step)
        parts = leaves[name].grad.double() * v
        # step^2 of third derivatives of order 1000 at most, 2^-50 / step, and fp32's sums
        assert abs(slope - float(parts.sum())) <= 2e-5 * float(parts.abs().sum()) + 1e-6, name


def test_in_a_graph():
    for shape, gate in (((3, 1024), (1024,)), ((8, 50, 300), (8, 1, 300))):
        o = make(shape, "bf16", 15, gate=gate)
        g = torch.randn(*shape, device=DEV).bfloat16()

        def step():
            r = ms.ops.residual_norm(**o, kind="layer")
            return [*r, *ms.ops.residual_norm_grad(g, None, r.residual, r.stats,
                                                   *(o[k] for k in NAMES[1:]), kind="layer")]

        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for seed in range(16, 20):
            o["residual"].copy_(make(shape, "bf16", seed)["residual"])
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_refusals():
    o = make((4, 8), "fp32", 21, gate=(8,))
    x, b, w = o["residual"], o["block"], o["weight"]
    call_ = ms.ops.residual_norm
    with pytest.raises(ValueError, match="kind|norm"):
        call_(x, b, w, kind="batch")
    with pytest.raises(ValueError, match="block"):
        call_(x, b[:3], w)
    with pytest.raises(TypeError, match="block"):
        call_(x, b.half(), w)
    with pytest.raises(ValueError, match="weight"):
        call_(x, b, w[:7])
    with pytest.raises(TypeError, match="weight"):
        call_(x, b, w.half())
    with pytest.raises(ValueError, match="bias"):
        call_(x, b, w, bias=w, kind="rms")
    with pytest.raises(ValueError, match="block_bias"):
        call_(x, b, w, block_bias=w, kind="layer")
    for bad in (w[:7], x[:, :7], x[:2], x.view(2, 2, 8)):
        with pytest.raises(ValueError, match="gate"):
            call_(x, b, w, gate=bad)
    y = x.view(2, 2, 8)
    with pytest.raises(ValueError, match="gate"):
        call_(y, b.view(2, 2, 8), w, gate=y[:1])
    with pytest.raises(ValueError, match="16384"):
        ms.ops.norm(torch.zeros(1, 16385, device=DEV), torch.zeros(16385, device=DEV))
    with pytest.raises(TypeError, match="residual"):
        ms.ops.norm(x.double(), w.double())
    with pytest.raises(RuntimeError, match="cpu"):
        call_(x, b.cpu(), w)
    with pytest.raises(RuntimeError, match="cpu"):
        call_(x, b, w.cpu())
    r = call_(x, b, w)
    grad = ms.ops.residual_norm_grad
    with pytest.raises(ValueError, match="None"):
        grad(None, None, r.residual, r.stats, b, w)
    with pytest.raises(ValueError, match="stats"):
        grad(x, None, r.residual, r.stats[:, :1], b, w)
    with pytest.raises(ValueError, match="stats"):
        grad(x, None, r.residual, r.stats, b, w, block_weight=w)
    with pytest.raises(ValueError, match="grad_out"):
        grad(x[:2], None, r.residual, r.stats, b, w)


def test_the_library_by_itself():
    lib = ctypes.CDLL(build.OPS_OUTPUT)
    P, I32, I64, F = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float
    lib.ms_norm_grad_workspace.restype = I64
    n, w = 90, 136
    o = make((n, w), "fp16", 22, "layer", True, (w,))
    p = {k: P(t.data_ptr()) for k, t in o.items()}
    rows = lambda t: ctypes.byref(Rows(t.data_ptr(), n, w, n, 0, w, 1, 0))  # noqa: E731
    nxt, out, stats = torch.empty_like(o["residual"]), torch.empty_like(o["residual"]), torch.empty(n, 4, device=DEV)
    stream = P(torch.cuda.current_stream().cuda_stream)
    assert lib.ms_norm(rows(o["residual"]), rows(o["block"]), I32(1), p["weight"], p["bias"],
                       p["block_weight"], p["block_bias"], p["gate"], I64(1), F(1), F(1e-5),
                       P(nxt.data_ptr()), P(out.data_ptr()), P(stats.data_ptr()), stream) == 0
    r = ms.ops.residual_norm(**o, kind="layer")
    assert torch.equal(nxt, r.residual) and torch.equal(out, r.out) and torch.equal(stats, r.stats)
    need = lib.ms_norm_grad_workspace(I64(n), I64(w), I32(1), I32(1), I32(1), I64(1))
    work = torch.full((need + 4096,), 77, dtype=torch.uint8, device=DEV)
    outs = [torch.empty_like(o[k]) for k in ("residual", "block", "weight", "bias", "block_weight",
                                             "block_bias", "gate")]
    g = torch.randn(n, w, device=DEV).half()
    assert lib.ms_norm_grad(rows(g), None, rows(nxt), P(stats.data_ptr()), rows(o["block"]), I32(1),
                            p["weight"], p["block_weight"], p["block_bias"], p["gate"], I64(1), F(1),
                            *(P(t.data_ptr()) for t in outs), P(work.data_ptr()), I64(need), stream) == 0
    assert bool((work[need:] == 77).all())
    want = ms.ops.residual_norm_grad(g, None, r.residual, r.stats, *(o[k] for k in NAMES[1:]), kind="layer")
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
