"""Activations held in 8 bits against their 64-bit definition.

Codes, exponents and the values that they stand for are compared exactly
(dividing by a power of two is exact, a code is one rounding).  An activation
carries the roundings of its exponential's argument (|argument| 2^-23 relative)
and a few more: 2^-21 (4 + |argument|) of the magnitudes of its terms, and half a
unit in the last place of the output.
"""

from __future__ import annotations

import math

import pytest
import torch
import torch.nn.functional as F
from torch.utils._python_dispatch import TorchDispatchMode

import minispeed_amd as ms
from tests import ops_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
KINDS = ["gelu", "gelu_tanh", "silu", "swiglu"]


def _rand(shape, dtype, seed, std=1.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * std
    x = x * torch.exp(torch.randn(shape[-1], generator=g) * 0.7) if shape else x
    return x.to(ref.DTYPES[dtype]).to(DEV)


def check_held(x):
    packed = ms.ops.pack8(x)
    codes, exponents, values = ref.held(x)
    assert packed.shape == tuple(x.shape) and packed.dtype == x.dtype
    assert torch.equal(packed.exponents.cpu(), exponents)
    assert torch.equal(packed.codes.cpu(), codes)
    assert packed.nbytes == codes.numel() + exponents.numel()
    back = ms.ops.unpack8(packed)
    assert back.shape == x.shape and back.dtype == x.dtype
    assert torch.equal(back.cpu().reshape(-1).nan_to_num(7.0, 8.0, 9.0),
                       values.to(x.dtype).nan_to_num(7.0, 8.0, 9.0))
    return values


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("shape", [(1,), (31,), (32,), (33,), (5, 7), (64, 64), (3, 1000), (2, 3, 129),
                                   (0,), (4, 0), (), (17, 257)])
def test_round_trip(dtype, shape):
    x = _rand(shape, dtype, 1)
    values = check_held(x)
    if x.numel():                                # within 1/127 of each block's largest
        flat = x.cpu().double().reshape(-1)
        most = torch.stack([b.abs().max().expand(len(b)) for b in flat.split(32)][:-1] or
                           [flat[:0]]).reshape(-1)
        most = torch.cat([most, flat[len(most):].abs().max().expand(len(flat) - len(most))])
        assert bool(((values - flat).abs() <= most / 127).all())


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_round_trip_of_edge_values(dtype):
    dt = ref.DTYPES[dtype]
    info = torch.finfo(dt)
    rows = []
    for top in (1.0, 127 / 128, 127.4 / 128, 127.5 / 128, 127.6 / 128, 255 / 256, 1.5, 2.0 ** -10,
                info.tiny, info.tiny * 3, info.smallest_normal / 2, info.max, info.max * 0.99,
                2.0 ** -24):
        row = torch.linspace(-1, 1, 32, dtype=torch.float64) * top
        row[3] = top
        row[4] = -0.0
        rows.append(row)
    x = torch.stack(rows).to(dt).to(DEV)
    check_held(x)
    check_held(torch.zeros(70, dtype=dt, device=DEV))
    for bad in (math.inf, -math.inf, math.nan):
        y = x.clone()
        y[2, 31], y[7, 0] = bad, bad
        check_held(y)
        back = ms.ops.unpack8(ms.ops.pack8(y))
        assert bool(torch.isnan(back[[2, 7]]).all()) and not bool(torch.isnan(back[[0, 1, 3, 6]]).any())


def test_round_trip_of_views():
    big = _rand((40, 130), "bf16", 2)
    for x in (big[:, 1:], big.t(), big[::2], big[:, ::3], big[:1].expand(9, 130), big.view(-1)[1:]):
        check_held(x)


def check_act(h, kind, up=None, grad_seed=3):
    a, saved = ms.ops.activation8(h, kind, up=up)
    assert a.shape == h.shape and a.dtype == h.dtype and a.is_contiguous()
    inputs = [h] if up is None else [h, up]
    held = []
    for x, s in zip(inputs, saved):
        codes, exponents, values = ref.held(x)
        assert torch.equal(s.codes.cpu(), codes) and torch.equal(s.exponents.cpu(), exponents)
        held.append(values.view(h.shape))
    f, _, scale, _ = ref.act(h.cpu(), kind)
    u = 1.0 if up is None else up.cpu().double()
    want = f * u
    ref.close(a, want, 2.0 ** -21 * scale * want.abs() + ref.rounding(want, h.dtype), f"{kind} a")

    grad = _rand(tuple(h.shape), {v: k for k, v in ref.DTYPES.items()}[h.dtype], grad_seed, 0.1)
    g = grad.cpu().double()
    grads, again = ms.ops.activation8_grad(saved, grad, kind)
    f, df, scale, size = ref.act(held[0], kind)
    u = torch.ones_like(f) if up is None else held[1]
    tol = 2.0 ** -21 * scale
    for got, want, terms in ((grads[0], g * u * df, (g * u).abs() * size),
                             (again, f * u, (f * u).abs())) + (
            () if up is None else ((grads[1], g * f, (g * f).abs()),)):
        assert got.shape == h.shape and got.dtype == h.dtype
        ref.close(got, want, tol * terms + ref.rounding(want, h.dtype), f"{kind} backward")
    assert len(grads) == len(inputs)
    less, none = ms.ops.activation8_grad(saved, grad, kind, again=False)
    assert none is None and all(torch.equal(x, y) for x, y in zip(less, grads))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("shape", [(1, 1), (3, 31), (8, 64), (5, 100), (2, 3, 256), (33, 1030),
                                   (0, 64), (130, 512)])
def test_activation(kind, dtype, shape):
    h = _rand(shape, dtype, 4)
    check_act(h, kind, _rand(shape, dtype, 5) if kind == "swiglu" else None)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_activation_over_its_range(kind, dtype):
    x = torch.cat([torch.linspace(-14, 14, 4001), torch.linspace(-0.01, 0.01, 799),
                   torch.tensor([0.0, -0.0, 1e-6, -1e-6, 40.0, -40.0, 200.0, -200.0, 30000.0,
                                 -30000.0])]).to(ref.DTYPES[dtype])
    if dtype != "fp16":
        x = torch.cat([x, torch.tensor([1e30, -1e30, 3e38, -3e38]).to(x.dtype)])
    # every value is alone in its block: it is held to one part in 64
    x = F.pad(x[:, None], (0, 31)).to(DEV)
    check_act(x, kind, torch.ones_like(x) if kind == "swiglu" else None)


@pytest.mark.parametrize("kind", KINDS)
def test_activation_in_32_bits_is_as_exact_as_its_operations(kind):
    """fp32: in units of 2^-24 of the terms, the exponential and the reciprocal are off by 2
    each, the exponential's argument (reduced to less than 1) and 1 + e by 1 each, the
    polynomial and what it is of by 4, and some 5 products and sums by 1 each: 16 at
    most, wherever the argument lies.  (gelu_tanh's argument is a product of its own, two
    roundings, which its exponential multiplies by its magnitude.)"""
    x = torch.cat([torch.linspace(-12.5, 12.5, 6001), torch.linspace(-0.05, 0.05, 800)]
                  + ([torch.linspace(-80, 80, 3001)] if kind in ("silu", "swiglu") else []))
    x = F.pad(x[:, None], (0, 31)).to(DEV)
    up = torch.ones_like(x) if kind == "swiglu" else None
    a, saved = ms.ops.activation8(x, kind, up=up)
    grads, again = ms.ops.activation8_grad(saved, torch.ones_like(x), kind)
    at = ref.held(x)[2].view(x.shape)
    for z, got_f, got_df in ((x.cpu().double(), a, None), (at, again, grads[0])):
        f, df, scale, size = ref.act(z, kind)
        unit = 2.0 ** -24 * (16 + (2 * scale if kind == "gelu_tanh" else 0))
        ref.close(got_f, f, unit * f.abs() + 2.0 ** -149, f"{kind} f")
        if got_df is not None:
            ref.close(got_df, df, unit * size + 2.0 ** -149, f"{kind} f'")


def test_activation_of_views():
    both = _rand((24, 2 * 96), "bf16", 6)
    gate, up = both.chunk(2, -1)
    check_act(gate, "swiglu", up)
    check_act(both[:, 1:97], "gelu")
    check_act(both[:, ::2], "silu")
    check_act(both.view(4, 6, 192)[:, 1:, 64:128], "gelu_tanh")
    check_act(both.view(4, 6, 192)[1:, ::2, :160].transpose(0, 1), "gelu")
    check_act(both[:1].expand(5, 192), "silu")
    odd = _rand((9, 2 * 33), "fp32", 7)
    check_act(odd[:, :33], "swiglu", odd[:, 33:])
    grad = both[:, :96].t().contiguous().t()
    _, saved = ms.ops.activation8(gate, "silu")
    assert torch.equal(ms.ops.activation8_grad(saved, grad, "silu")[0][0],
                       ms.ops.activation8_grad(saved, grad.contiguous(), "silu")[0][0])


def test_overflow_reaches_the_gradient():
    h = _rand((4, 64), "fp16", 8)
    h[1, 5] = math.inf
    a, saved = ms.ops.activation8(h, "gelu")
    (dh,), again = ms.ops.activation8_grad(saved, torch.ones_like(h), "gelu")
    assert bool(torch.isnan(dh[1, :32]).all()) and bool(torch.isnan(again[1, :32]).all())
    rest = torch.cat([dh[0], dh[1, 32:], dh[2:].reshape(-1)])
    assert bool(torch.isfinite(rest).all()) and torch.isinf(a[1, 5])


def test_past_32_bits():
    n = 2 ** 32 + 96                             # 8.6 GB
    x = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    x[-40:] = 1.75
    x[5] = -3.0
    held = ms.ops.pack8(x)
    back = ms.ops.unpack8(held)
    assert bool((back[-40:] == 1.75).all()) and back[5] == -3.0
    assert int(torch.count_nonzero(back[6:-40])) == 0
    del back, held
    a, saved = ms.ops.activation8(x.view(-1, 32), "silu")
    assert bool((a.view(-1)[-40:] == F.silu(x[-40:].float()).bfloat16()).all())
    assert int(torch.count_nonzero(a.view(-1)[6:-40])) == 0
    (dh,), a = ms.ops.activation8_grad(saved, x.view(-1, 32), "silu")
    assert int(torch.count_nonzero(dh.view(-1)[6:-40])) == 0 and dh.view(-1)[-1] > 1.75


@pytest.mark.parametrize("kind", KINDS)
def test_activation_linear_autograd(kind):
    n, f, d = 24, 160, 48
    h = _rand((2, n // 2, f), "fp32", 9).requires_grad_()
    up = _rand((2, n // 2, f), "fp32", 10).requires_grad_() if kind == "swiglu" else None
    w = _rand((d, f), "fp32", 11, 0.1).requires_grad_()
    b = _rand((d,), "fp32", 12, 0.1).requires_grad_()
    y = ms.ops.activation8_linear(h, w, b, kind, up)
    ref_a = ref.act(h.detach().cpu(), kind)[0] * (1 if up is None else up.detach().cpu().double())
    want = ref_a.reshape(n, f) @ w.detach().cpu().double().t() + b.detach().cpu().double()
    assert torch.allclose(y.detach().cpu().double().view(n, d), want, rtol=1e-4, atol=1e-4)
    gy = _rand((2, n // 2, d), "fp32", 13)
    y.backward(gy)
    # the 64-bit backward pass at the held values
    hv = ref.held(h)[2].view(n, f).requires_grad_()
    uv = None if up is None else ref.held(up)[2].view(n, f).requires_grad_()
    wv = w.detach().cpu().double().requires_grad_()
    base = 0.5 * hv * torch.special.erfc(-hv / math.sqrt(2.0)) if kind == "gelu" else (
        F.gelu(hv, approximate="tanh") if kind == "gelu_tanh" else F.silu(hv))
    ((base * (1 if uv is None else uv)) @ wv.t()).backward(gy.cpu().double().view(n, d))
    for got, exact in ((h.grad, hv.grad), (w.grad, wv.grad)) + (
            () if up is None else ((up.grad, uv.grad),)):
        assert torch.allclose(got.cpu().double().reshape(exact.shape), exact, rtol=1e-4,
                              atol=1e-4 * float(exact.abs().max()))
    assert torch.allclose(b.grad.cpu().double(), gy.cpu().double().view(n, d).sum(0), rtol=1e-4, atol=1e-4)
    # against differences of the 64-bit form in one direction
    v = torch.randn(n, f, generator=torch.Generator().manual_seed(14), dtype=torch.float64)

    def loss(z):
        a = ref.act(z, kind)[0] * (1 if uv is None else uv.detach())
        return float(((a @ wv.detach().t()) * gy.cpu().double().view(n, d)).sum())

    step = 1e-5
    slope = (loss(hv.detach() + step * v) - loss(hv.detach() - step * v)) / (2 * step)
    prod = h.grad.cpu().double().view(n, f) * v
    assert abs(slope - float(prod.sum())) <= 1e-4 * float(prod.abs().sum())


@pytest.mark.parametrize("kind", KINDS)
def test_activation_autograd(kind):
    """The activation's gradients are those of its backward pass, for whichever inputs want them."""
    h0, g = _rand((3, 70), "bf16", 25), _rand((3, 70), "bf16", 27, 0.1)
    up0 = _rand((3, 70), "bf16", 26) if kind == "swiglu" else None
    plain, saved = ms.ops.activation8(h0, kind, up=up0)
    grads, _ = ms.ops.activation8_grad(saved, g, kind)
    for want_h, want_up in ((True, True), (True, False), (False, True)):
        h, up = h0.clone().requires_grad_(want_h), None
        if kind == "swiglu":
            up = up0.clone().requires_grad_(want_up)
        elif not want_h:
            continue
        a, held = ms.ops.activation8(h, kind, up=up)
        assert a.requires_grad and torch.equal(a.detach(), plain)
        assert all(torch.equal(x.codes, y.codes) and torch.equal(x.exponents, y.exponents)
                   and not x.codes.requires_grad for x, y in zip(held, saved))
        a.backward(g)
        assert torch.equal(h.grad, grads[0]) if want_h else h.grad is None
        if up is not None:
            assert torch.equal(up.grad, grads[1]) if want_up else up.grad is None
    with torch.no_grad():
        assert not ms.ops.activation8(h, kind, up=up)[0].requires_grad


class _Products(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.n = 0

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.n += func.overloadpacket in (torch.ops.aten.mm, torch.ops.aten.addmm, torch.ops.aten.bmm)
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize("kind", ["gelu", "swiglu"])
def test_activation_linear_computes_no_product_that_nobody_wants(kind):
    h, w0 = _rand((2, 9, 64), "bf16", 28), _rand((32, 64), "bf16", 29, 0.1)
    up = _rand((2, 9, 64), "bf16", 30) if kind == "swiglu" else None
    gy, got = _rand((2, 9, 32), "bf16", 31), {}
    for want_h, want_w, products in ((True, True, 2), (False, True, 1), (True, False, 1)):
        x, w = h.clone().requires_grad_(want_h), w0.clone().requires_grad_(want_w)
        y = ms.ops.activation8_linear(x, w, None, kind, up)
        # the backward pass runs in autograd's own thread: called here for the mode to see it
        node, count = y.grad_fn, _Products()
        with count, torch.no_grad():
            grads = type(node)._forward_cls.backward(node, gy)
        assert count.n == products, (want_h, want_w, count.n)
        y.backward(gy)
        for name, t, g in (("h", x, grads[0]), ("w", w, grads[2])):
            if t.requires_grad:
                assert torch.equal(t.grad, got.setdefault(name, t.grad)) and torch.equal(t.grad, g)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("half_h", [False, True])
def test_activation_linear_under_autocast(dtype, half_h):
    """fp32 parameters, products in half precision: a product of 64 terms is off by
    at most a rounding of each operand, the sum and the result (2^-8 for bf16)."""
    kind, n, f, d = "silu", 24, 64, 48
    w, b = _rand((d, f), "fp32", 17, 0.1).requires_grad_(), _rand((d,), "fp32", 18).requires_grad_()
    h0 = _rand((n, f), dtype if half_h else "fp32", 19)
    gy = _rand((n, d), dtype, 20)
    h = h0.clone().requires_grad_()
    with torch.autocast("cuda", ref.DTYPES[dtype]):
        y = ms.ops.activation8_linear(h, w, b, kind)
    y.backward(gy)
    assert y.dtype == gy.dtype and h.grad.dtype == h.dtype
    assert w.grad.dtype == b.grad.dtype == torch.float32
    hv = ref.held(h0)[2].view(n, f).requires_grad_()
    wv = w.detach().cpu().double().requires_grad_()
    (F.silu(hv) @ wv.t()).backward(gy.cpu().double())
    unit = 2.0 ** (-11 if dtype == "fp16" else -8)
    size = (gy.cpu().double().abs() @ wv.detach().abs()) * 1.1
    assert bool(((h.grad.cpu().double() - hv.grad).abs() <= 5 * unit * size).all())
    size = gy.cpu().double().abs().t() @ F.silu(hv.detach()).abs()
    assert bool(((w.grad.cpu().double() - wv.grad).abs() <= 5 * unit * size + 1e-6).all())


def test_checkpoint_of_a_host_tensor():
    x, host = _rand((4, 32), "fp32", 21).requires_grad_(), torch.arange(4.0)
    ms.ops.checkpoint8(lambda z, c: (z * c.to(DEV)[:, None]).sum(), x, host).backward()
    assert torch.equal(x.grad, host.to(DEV)[:, None].expand(4, 32))


def test_checkpoint_runs_again_on_the_held_values():
    torch.manual_seed(0)
    layer = torch.nn.Sequential(torch.nn.Linear(64, 96), torch.nn.GELU(), torch.nn.Dropout(0.5),
                                torch.nn.Linear(96, 64)).to(DEV)
    x = _rand((10, 64), "fp32", 15).requires_grad_()
    ids = torch.arange(10, device=DEV)
    seen = []

    def fn(z, ids, factor, other=None):
        seen.append(z.detach().clone())
        return layer(z) * factor, (z * ids[:, None]).sum()

    state = torch.cuda.get_rng_state()
    y, s = ms.ops.checkpoint8(fn, x, ids, 2.0, None)
    after = torch.cuda.get_rng_state()
    (y.sum() + s).backward()
    assert torch.equal(torch.cuda.get_rng_state(), after)
    assert torch.equal(seen[0], x.detach()) and torch.equal(
        seen[1].cpu().double().reshape(-1), ref.held(x)[2])
    got = [x.grad.clone()] + [p.grad.clone() for p in layer.parameters()]
    # the same by hand: the second run at the held values with the same numbers
    for p in layer.parameters():
        p.grad = None
    z = seen[1].clone().requires_grad_()
    torch.cuda.set_rng_state(state)
    y, s = fn(z, ids, 2.0)
    (y.sum() + s).backward()
    for a, b in zip(got, [z.grad] + [p.grad for p in layer.parameters()]):
        assert torch.equal(a, b)


def test_checkpoint_of_half_precision_and_of_nothing():
    w = _rand((32, 32), "bf16", 16).requires_grad_()
    x = _rand((8, 32), "bf16", 17).requires_grad_()
    y = ms.ops.checkpoint8(lambda a, b: a @ b, x, w)
    y.backward(torch.ones_like(y))
    held = ms.ops.unpack8(ms.ops.pack8(x.detach()))
    assert torch.equal(w.grad, held.t() @ torch.ones_like(y))
    assert x.grad.dtype == torch.bfloat16
    assert not ms.ops.checkpoint8(lambda a: a * 2, x.detach()).requires_grad


def test_checkpoint_keeps_masks_tables_and_parameters_as_they_are():
    torch.manual_seed(1)
    x = _rand((2, 12, 32), "fp32", 22).requires_grad_()
    mask = torch.full((12, 12), -math.inf, device=DEV).triu(1)
    table = _rand((12, 32), "fp32", 23)
    w = torch.nn.Parameter(_rand((32, 32), "fp32", 24, 0.1))
    seen = []

    def fn(z, mask, table, w):
        seen.append((mask.detach().clone(), table.detach().clone(), w.detach().clone()))
        return torch.softmax((z * table) @ z.transpose(1, 2) + mask, -1) @ (z @ w)

    y = ms.ops.checkpoint8(fn, x, mask, table, w)
    y.backward(torch.ones_like(y))
    for a, b in zip(*seen):
        assert torch.equal(a, b)
    z, v = x.detach().clone(), w.detach().clone().requires_grad_()
    z = ref.held(z)[2].view(z.shape).float().to(DEV).requires_grad_()
    fn(z, mask, table, v).backward(torch.ones_like(y))
    assert torch.equal(x.grad, z.grad) and torch.equal(w.grad, v.grad)
    assert bool(torch.isfinite(x.grad).all()) and bool(x.grad.any())


def test_in_a_graph():
    h, up, g = (_rand((40, 200), "bf16", s) for s in (18, 19, 20))

    def step():
        a, saved = ms.ops.activation8(h, "swiglu", up=up)
        grads, again = ms.ops.activation8_grad(saved, g, "swiglu")
        return [a, *grads, again, ms.ops.unpack8(ms.ops.pack8(h))]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(21, 25):
        h.copy_(_rand((40, 200), "bf16", seed))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_refusals():
    x = _rand((4, 64), "fp32", 26)
    a, saved = ms.ops.activation8(x, "gelu")
    _, two = ms.ops.activation8(x, "swiglu", up=x)
    with pytest.raises(ValueError, match="unknown activation"):
        ms.ops.activation8(x, "relu")
    with pytest.raises(ValueError, match="gated"):
        ms.ops.activation8(x, "gelu", up=x)
    with pytest.raises(ValueError, match="gated"):
        ms.ops.activation8(x, "swiglu")
    with pytest.raises(ValueError, match="up"):
        ms.ops.activation8(x, "swiglu", up=x[:2])
    with pytest.raises(TypeError, match="up"):
        ms.ops.activation8(x, "swiglu", up=x.half())
    with pytest.raises(TypeError, match="dtype"):
        ms.ops.activation8(x.double(), "gelu")
    with pytest.raises(TypeError, match="dtype"):
        ms.ops.pack8(x.long())
    with pytest.raises(RuntimeError, match="cpu"):
        ms.ops.pack8(x.cpu())
    with pytest.raises(ValueError, match="checkpoint"):
        ms.ops.activation8_grad(saved, x.half(), "gelu")
    with pytest.raises(ValueError, match="checkpoint"):
        ms.ops.activation8_grad(saved, x[:2], "gelu")
    with pytest.raises(ValueError, match="checkpoint"):
        ms.ops.activation8_grad(saved, x, "swiglu")
    with pytest.raises(ValueError, match="checkpoint"):
        ms.ops.activation8_grad(two, x, "gelu")
    with pytest.raises(ValueError, match="checkpoint"):
        ms.ops.activation8_grad((), x, "gelu")
    with pytest.raises(ValueError, match="hold"):
        ms.ops.unpack8(ms.ops.Checkpoint8(saved[0].codes, saved[0].exponents, (4, 63), x.dtype))
    with pytest.raises(TypeError, match="dtype"):
        ms.ops.unpack8(ms.ops.Checkpoint8(saved[0].codes, saved[0].exponents, (4, 64), torch.int32))
