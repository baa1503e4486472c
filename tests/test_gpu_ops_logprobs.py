"""Log probabilities, entropy, alternatives and the logits' gradient against
64-bit sums.

Tolerances.  A term 2^y of the sum carries the rounding of y (|y| 2^-24) and of
the exponential (2^-22); terms are added at most V / 64 + 64 in a row, 2^-24
each: rel = 2^-24 (V / 64 + 96 + 2 spread), with spread the largest |x - max| that
still counts (32: the rest adds less than 2^-46).  The logarithm of the sum is
off by rel, and lse and logprob by their own roundings and those of the
products with log2 e: 2^-22 of the magnitudes that meet there.  The entropy is
log s - t / s, each off by rel of its magnitudes.
"""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import minispeed_amd as ms
from minispeed_amd import build
from tests import ops_reference as ref
from tests.test_ops_abi import Rows, Tokens

pytestmark = pytest.mark.gpu
DEV = "cuda"
INF, NAN = math.inf, math.nan


def _logits(n, v, dtype, seed, std=2.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, v, generator=g) * std).to(ref.DTYPES[dtype]).to(DEV)


def _targets(n, v, seed, ignored=0.2):
    g = torch.Generator().manual_seed(seed)
    t = torch.randint(0, v, (n,), generator=g)
    t[torch.rand(n, generator=g) < ignored] = -100
    return t.to(DEV)


def _tolerances(logits, targets, want):
    v = logits.shape[-1]
    rel = 2.0 ** -24 * (v / 64 + 96 + 64)
    x = logits.double().cpu()
    t = targets.cpu().long().clamp(0, v - 1)
    given = x.gather(-1, t[..., None])[..., 0].abs().nan_to_num(0, 0, 0)
    lse = want["lse"].abs().nan_to_num(0, 0, 0)
    ent = want["entropy"].abs().nan_to_num(0, 0, 0)
    logp = want["logprob"].abs().nan_to_num(0, 0, 0)
    return {"lse": rel + 2.0 ** -22 * lse,
            "logprob": rel + 2.0 ** -22 * (given + lse.clamp(max=1024.0) + logp),
            "entropy": rel * (4 + 2 * ent) * 2,
            "top_logprob": (rel + 2.0 ** -22 * (2 * lse.clamp(max=1024.0) + 64))[..., None]
            + 2.0 ** -22 * want["top_logprob"].abs().nan_to_num(0, 0, 0)}


def check(logits, targets, top=0, entropy=True, ignore_index=-100):
    got = ms.ops.token_logprobs(logits, targets, top=top, entropy=entropy,
                                ignore_index=ignore_index)
    want = ref.logprobs(logits, targets, top, ignore_index)
    tol = _tolerances(logits, targets, want)
    names = ["logprob", "lse"] + ["entropy"] * entropy + ["top_logprob"] * bool(top)
    for name in names:
        value = getattr(got, name)
        assert value.dtype == torch.float32 and value.shape == want[name].shape
        ref.close(value, want[name], tol[name], f"{name} {tuple(logits.shape)} {logits.dtype}")
    if top:
        assert got.top_id.dtype == torch.int64
        assert torch.equal(got.top_id.cpu(), want["top_id"])
    else:
        assert got.top_logprob is None and got.top_id is None
    assert entropy or got.entropy is None
    return got


def check_grad(logits, targets, entropy=True, seed=0, ignore_index=-100):
    gen = torch.Generator().manual_seed(seed)
    g = torch.randn(targets.shape, generator=gen).to(DEV)
    h = (torch.randn(targets.shape, generator=gen) * 0.1).to(DEV) if entropy else None
    r = ms.ops.token_logprobs(logits, targets, entropy=entropy, ignore_index=ignore_index)
    got = ms.ops.token_logprobs_grad(logits, targets, r.lse, g, r.entropy, h, ignore_index)
    assert got.shape == logits.shape and got.dtype == logits.dtype
    want, size = ref.logprobs_grad(logits, targets, g, h, ignore_index)
    lse = r.lse.double().cpu().abs().nan_to_num(0, 0, 0)[..., None].clamp(max=1024.0)
    x = logits.double().cpu().abs().nan_to_num(0, 0, 0).clamp(max=1024.0)
    # p carries the roundings of x L and lse L and lse's own error, log p + entropy
    # those of both: relative to the terms' magnitudes
    v = logits.shape[-1]
    rel = 2.0 ** -22 * (lse + x + 16) + 2 * 2.0 ** -24 * (v / 64 + 160)
    p_floor = 2.0 ** -126                    # below, exponentials may be flushed to zero
    extra = (g.double().cpu().abs()[..., None] + (0 if h is None else
             h.double().cpu().abs()[..., None] * 200)) * p_floor
    # the entropy's error times p h
    if h is not None:
        extra = extra + h.double().cpu().abs()[..., None] * torch.softmax(
            logits.double().cpu(), -1).nan_to_num(0) * rel * 32
    ref.close(got, want, size * rel + extra + ref.rounding(want, logits.dtype),
              f"grad {tuple(logits.shape)} {logits.dtype}")
    return got


SIZES = [(1, 1), (3, 2), (2, 7), (5, 63), (4, 65), (7, 512), (3, 1000), (2, 4097), (3, 50257),
         (1, 50257), (2, 128256), (1, 262145), (130, 777)]


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("n,v", SIZES)
def test_logprobs(dtype, n, v):
    x, t = _logits(n, v, dtype, 1), _targets(n, v, 2)
    check(x, t, top=0, entropy=False)
    check(x, t, top=min(v, 5))
    check(x, t, top=min(v, 64), entropy=False)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("n,v", SIZES)
def test_grad(dtype, n, v):
    x, t = _logits(n, v, dtype, 3), _targets(n, v, 4)
    check_grad(x, t, entropy=False)
    check_grad(x, t, entropy=True)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("v", [64, 250, 300, 600, 1030, 2048, 4090, 4096])
def test_short_rows(v, dtype):
    """Rows that a wave holds: any contents, orders and starts."""
    n, low = 24, torch.finfo(ref.DTYPES[dtype]).min
    wide = _logits(n, v + 3, dtype, 51)
    x = wide[:, 3:]                               # rows 3 values off, one after the other
    ramp = torch.linspace(-4, 4, v).to(x.dtype).to(DEV)
    x[1], x[2], x[3] = ramp, ramp.flip(0), (torch.arange(v, device=DEV) % 3).to(x.dtype)
    x[4], x[5], x[6] = -INF, low, 0.0
    x[7, 5:], x[8, 5:], x[9, : v - 5] = -INF, low, -1e4
    x[10], x[11] = torch.finfo(x.dtype).max / 2, -3000.0
    x[12, v // 2], x[13, v // 3], x[14] = INF, NAN, NAN
    x[15] = torch.where(torch.arange(v, device=DEV) // 64 == 2, 5.0 + ramp.float(), -1.0).to(x.dtype)
    t = _targets(n, v, 52)
    for top in (0, 1, 20, min(v, 64)):
        check(x, t, top=top, entropy=top != 20)
    good = [r for r in range(n) if r not in (12, 13, 14)]
    check_grad(x[good], t[good])
    check_grad(wide[:12, 3:], t[:12], entropy=False)


def test_more_short_rows_than_waves():
    x, t = _logits(20_000, 40, "bf16", 53), _targets(20_000, 40, 54)
    check(x, t, top=3)
    check_grad(x, t)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_many_rows(dtype):
    x, t = _logits(2100, 1030, dtype, 5), _targets(2100, 1030, 6)
    check(x, t, top=3)
    check_grad(x, t)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_layouts(dtype):
    b, t, v = 3, 9, 517
    big = _logits(b * t, v + 5, dtype, 7).view(b, t, v + 5)
    ids = _targets(b * (t + 1), v, 8).view(b, t + 1)
    for x, y in ((big[:, :-1, :v], ids[:, 1:-1]), (big[:, :, 2:v + 2], ids[:, 1:]),
                 (big[..., 5:].transpose(0, 1), ids[:, 1:].t()), (big[:, :, ::2], ids[:, 1:] // 2),
                 (big[:, :1, 1:v + 1].expand(b, t, v), ids[:, :-1].int()),
                 (big[1, 2, :v], ids[1, 2]), (big[:0, :, :v], ids[:0, 1:]),
                 (big[:, :, :v].reshape(1, b, t, v)[:, :, 1:], ids[None, :, 2:])):
        y = torch.where(y < 0, torch.full_like(y, -100), y)
        check(x, y, top=4)
        check_grad(x, y)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("v", [33, 5000, 50257])
def test_masks(dtype, v):
    x, t = _logits(12, v, dtype, 9), _targets(12, v, 10, 0.0)
    low = torch.finfo(x.dtype).min
    x[:, 1::3] = -INF
    x[1] = -INF                                  # nothing left
    x[2] = low                                   # all masked by the type's lowest value
    x[3, 5:] = low
    x[4] = -INF
    x[4, v - 1] = 1.5                            # one left, and it is the last
    x[5] = 0.0                                   # all equal
    x[6] = -0.0
    x[6, ::2] = 0.0
    x[7] = torch.finfo(x.dtype).max / 2
    x[8, v // 2] = torch.finfo(x.dtype).max
    x[9] = -3000.0
    x[9, 7] = -2990.0
    x[10, 1:] = -INF
    x[11] = low
    x[11, ::2] = -INF
    t[4], t[10] = v - 1, 0
    check(x, t, top=min(v, 20))
    check_grad(x, t)
    check_grad(x, t, entropy=False)


@pytest.mark.parametrize("n", [3, 257])             # rows that are split, and that are not
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_masked_stretches(dtype, n):
    """A mask that leaves the last values, one in the middle, or a few."""
    v = 33_000
    low = torch.finfo(ref.DTYPES[dtype]).min
    for fill in (-INF, low, -1e4, -70.0, -6e5 if dtype != "fp16" else -6e4):
        x, t = _logits(n, v, dtype, 41), _targets(n, v, 42)
        x[0, :-5] = fill
        x[1, :20_000] = fill
        x[2, : v // 2], x[2, v // 2 + 1:] = fill, fill
        if n > 3:
            x[3:9, torch.arange(v, device=DEV) % 3001 != 17] = fill
            x[9, : v // 2], x[9, v // 2:] = low, fill
            x[10] = fill
            x[10, ::2] = fill - 1 if -1e6 < fill else fill
        check(x, t, top=8)
        check(x, t, entropy=False)
        check_grad(x, t)


@pytest.mark.parametrize("n", [2, 257])
@pytest.mark.parametrize("above", [60.0, 68.0, 75.0, 84.0, 86.0, 88.0, 89.0, 300.0])
def test_one_far_above_the_others(above, n):
    v = 50_257
    x = _logits(n, v, "fp32", 43)
    x[:, 40_000] = above
    x[0, -1] = above
    t = torch.full((n,), 40_000, device=DEV)
    check(x, t, top=3)
    check(x, t)


def test_nan_and_infinity():
    v = 700
    x, t = _logits(6, v, "fp32", 11), _targets(6, v, 12, 0.0)
    x[0, 3] = NAN
    x[1, 699] = INF
    x[2] = NAN
    x[3, 4], x[3, 5], x[3, 600] = INF, NAN, NAN
    x[4] = -INF
    x[4, 8] = NAN
    check(x, t, top=7)
    r = ms.ops.token_logprobs(x, t, entropy=True)
    one = torch.ones(6, device=DEV)
    d = ms.ops.token_logprobs_grad(x, t, r.lse, one, r.entropy, one)
    assert bool(torch.isnan(d[:5]).all()) and bool(torch.isfinite(d[5]).all())


@pytest.mark.parametrize("v", [65, 4096, 50257])
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_gradient_of_nan_logits_beside_an_empty_lse(dtype, v):
    """A row whose lse says that nothing is left, and a NaN that has come into it since."""
    x = torch.full((3, v), -INF, dtype=ref.DTYPES[dtype], device=DEV)
    x[0, v // 2], x[1] = NAN, NAN
    lse, one = torch.full((3,), -INF, device=DEV), torch.ones(3, device=DEV)
    t = torch.zeros(3, dtype=torch.int64, device=DEV)
    for h in (None, one):
        d = ms.ops.token_logprobs_grad(x, t, lse, one, one, h)
        assert torch.equal(torch.isnan(d), torch.isnan(x))
        assert not bool(d.nan_to_num(0.0).any())


# a few values more than a whole number of blocks of the gradient (2048 values of 2 bytes,
# 1024 of 4), in rows that begin anywhere within 16 bytes
@pytest.mark.parametrize("dtype,v", [("fp32", 2049), ("fp32", 4097), ("fp32", 4098), ("fp16", 4097),
                                     ("bf16", 4102), ("bf16", 8193), ("fp16", 32769)])
def test_gradient_of_odd_rows_between_others(dtype, v):
    """Rows with nothing left and rows far from 0 before ordinary ones and at the end."""
    x, t = _logits(17, v, dtype, 61), _targets(17, v, 62)
    x[1::4] = -INF
    x[3::4] = (x[3::4].float() - 3000.0).to(x.dtype)
    x[16] = -INF
    check_grad(x, t)
    check_grad(x, t, entropy=False)
    x[16] = (_logits(1, v, dtype, 63)[0].float() + 900.0).to(x.dtype)
    check_grad(x, t)


@pytest.mark.parametrize("dtype,v", [("fp32", 2049), ("bf16", 4097), ("fp16", 8193)])
@pytest.mark.parametrize("fill", [-INF, -3000.0])
def test_gradient_stays_within_its_rows(dtype, v, fill):
    """What lies before and behind the gradient is not written, and what lies before and
    behind the logits is not used."""
    n, edge = 9, 64
    whole = torch.full((n * v + 2 * edge,), NAN, dtype=ref.DTYPES[dtype], device=DEV)
    x = whole[edge:-edge].view(n, v).fill_(fill)
    out = torch.full_like(whole, 7.0)
    t = torch.zeros(n, dtype=torch.int64, device=DEV)
    lse, g = torch.logsumexp(x.float(), 1), torch.ones(n, device=DEV)
    lib = ctypes.CDLL(build.OPS_OUTPUT)
    rows = Rows(x.data_ptr(), n, v, n, 0, v, ["fp32", "fp16", "bf16"].index(dtype), 0)
    ids = Tokens(t.data_ptr(), n, n, 0, 1, 1, 0)
    ptr = ctypes.c_void_p
    assert lib.ms_logprobs_grad(ctypes.byref(rows), ctypes.byref(ids), ctypes.c_int64(-100),
                                ptr(lse.data_ptr()), None, ptr(g.data_ptr()), None,
                                ptr(out[edge:].data_ptr()),
                                ptr(torch.cuda.current_stream().cuda_stream)) == 0
    assert bool((out[:edge] == 7.0).all()) and bool((out[-edge:] == 7.0).all())
    d = out[edge:-edge].view(n, v).float()
    p = 0.0 if fill == -INF else 1.0 / v
    assert torch.allclose(d[:, 1:], torch.full_like(d[:, 1:], -p), rtol=0.01, atol=0.0)
    assert torch.allclose(d[:, 0], torch.full_like(d[:, 0], 1.0 - p if p else 0.0), rtol=0.01)


def test_gradient_of_rows_far_from_zero_is_no_order_slower():
    """Logits that share a large offset cost a pass more, not one for every block of a row."""
    n, v = 2048, 50257
    near, t = _logits(n, v, "bf16", 64), _targets(n, v, 65)
    far = (near.float() + 4096.0).to(near.dtype)
    g, us = torch.ones(n, device=DEV), []
    for x in (near, far):
        lse = ms.ops.token_logprobs(x, t).lse
        times = []
        for _ in range(5):
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            start.record()
            ms.ops.token_logprobs_grad(x, t, lse, g)
            end.record()
            end.synchronize()
            times.append(start.elapsed_time(end))
        us.append(min(times))
    assert us[1] < 8 * us[0], us


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_alternatives_of_short_rows_with_little_left(dtype):
    """Rows that a mask leaves nothing, or less than there are alternatives: the first
    indices of what is masked follow, in a pass or two over the row."""
    n, v = 8, 3001
    plain, t = _logits(n, v, dtype, 66), _targets(n, v, 67)
    x = plain.clone()
    x[3], x[4, 7:], x[5, : v - 9] = -INF, -INF, torch.finfo(x.dtype).min
    x[6], x[7, ::2] = -1.5, -INF
    for top in (1, 4, 5, 7, 8, 20, 64):
        check(x, t, top=top)
    us = []
    for z in (plain, x):
        times = []
        for _ in range(20):
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            start.record()
            ms.ops.token_logprobs(z, t, top=5)
            end.record()
            end.synchronize()
            times.append(start.elapsed_time(end))
        us.append(1e3 * min(times))
    assert us[1] < us[0] + 60.0, us


def test_targets_outside_the_vocabulary():
    x = _logits(5, 100, "bf16", 13)
    t = torch.tensor([100, -1, 7, 2 ** 40, -100], device=DEV)
    check(x, t, top=1)
    r = ms.ops.token_logprobs(x, t)
    d = ms.ops.token_logprobs_grad(x, t, r.lse, torch.ones(5, device=DEV))
    assert bool(torch.isnan(d[[0, 1, 3]]).all()) and bool(torch.isfinite(d[2]).all())
    assert not bool(d[4].any())
    check(x, torch.tensor([7, 3, 7, 9, 7], device=DEV), ignore_index=7)


@pytest.mark.parametrize("order", ["rising", "falling", "steps", "lump"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_alternatives_of_ordered_rows(order, dtype):
    v = 20_011
    ramp = torch.linspace(-4, 4, v)
    x = {"rising": ramp, "falling": ramp.flip(0), "steps": (torch.arange(v) % 3).float(),
         "lump": torch.where((torch.arange(v) // 64) == 100, 5.0 + ramp, -1.0)}[order]
    x = torch.stack([x, x.roll(777)]).to(ref.DTYPES[dtype]).to(DEV)
    for top in (1, 20, 64):
        check(x, torch.zeros(2, dtype=torch.int64, device=DEV), top=top)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_many_places_to_look_again(dtype):
    """Two far apart places of many threads hold what may be an alternative."""
    n, v, apart = 257, 131072, 65536
    x = _logits(n, v, dtype, 31, std=1.0)
    high = torch.arange(0, 800, 8)
    for start in (0, apart):
        values = 8 + torch.randn(n, len(high), generator=torch.Generator().manual_seed(start))
        x[:, (high + start).to(DEV)] = values.to(x.dtype).to(DEV)
    check(x, _targets(n, v, 32), top=50)


def test_rows_past_32_bits():
    n, v = 17_000, 131_072                        # 2.2e9 values, 4.5 GB
    x = torch.zeros(n, v, dtype=torch.bfloat16, device=DEV)
    x[-1, -1] = 8.0
    t = torch.full((n,), v - 1, device=DEV)
    r = ms.ops.token_logprobs(x, t, top=1)
    want = -math.log1p((v - 1) * math.exp(-8.0))
    assert abs(float(r.logprob[-1]) - want) <= 1e-5 and int(r.top_id[-1, 0]) == v - 1
    assert torch.allclose(r.logprob[:-1], torch.tensor(-math.log(v), device=DEV), rtol=1e-6)
    assert not bool(r.top_id[:-1].any())
    d = ms.ops.token_logprobs_grad(x, t, r.lse, torch.ones(n, device=DEV))
    assert abs(float(d[-1, -1]) - (1 - math.exp(want))) <= 0.01
    assert abs(float(d[-2, -1]) - 1) <= 0.01 and abs(float(d[-1, 0]) * v + v * math.exp(want - 8)) <= 0.1


def test_the_same_bits_every_time_and_on_another_stream():
    x, t = _logits(70, 50257, "fp16", 14), _targets(70, 50257, 15)
    first = ms.ops.token_logprobs(x, t, top=9, entropy=True)
    g = torch.ones(70, device=DEV)
    grad = ms.ops.token_logprobs_grad(x, t, first.lse, g, first.entropy, g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(side):
            again = ms.ops.token_logprobs(x, t, top=9, entropy=True)
            d = ms.ops.token_logprobs_grad(x, t, again.lse, g, again.entropy, g)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, again)) and torch.equal(d, grad)


def test_autograd_against_the_formula_and_differences():
    n, v = 6, 301
    x = _logits(n, v, "fp32", 16).requires_grad_()
    t = _targets(n, v, 17)
    r = ms.ops.token_logprobs(x, t, top=3, entropy=True)
    assert r.logprob.requires_grad and r.entropy.requires_grad
    assert not (r.lse.requires_grad or r.top_logprob.requires_grad or r.top_id.requires_grad)
    (r.logprob.sum() * -0.5 + 0.25 * r.entropy.mean()).backward()
    d, size = ref.logprobs_grad(x, t, torch.full((n,), -0.5), torch.full((n,), 0.25 / n))
    ref.close(x.grad, d, size * 2.0 ** -17 + 2.0 ** -40)

    def loss(z):
        w = ref.logprobs(z, t, 0)
        return float(w["logprob"].sum() * -0.5 + 0.25 * w["entropy"].mean())

    # central differences of the 64-bit loss: error step^2 / 6 of the third
    # derivative (below 4 per row here, the direction's entries below 5) and
    # 2^-50 / step
    direction = _logits(n, v, "fp32", 18, 1.0).double()
    step = 1e-5
    slope = (loss(x.detach().double() + step * direction)
             - loss(x.detach().double() - step * direction)) / (2 * step)
    got = float((x.grad.double() * direction).sum())
    assert abs(slope - got) <= 1e-5 * float((x.grad.double() * direction).abs().sum()) + 1e-8
    # one output alone
    x.grad = None
    ms.ops.token_logprobs(x, t, entropy=True).entropy.sum().backward()
    d, size = ref.logprobs_grad(x, t, None, torch.ones(n))
    ref.close(x.grad, d, size * 2.0 ** -17 + 2.0 ** -40)
    assert not ms.ops.token_logprobs(x.detach(), t).logprob.requires_grad


def test_in_a_graph():
    for n, v in ((3, 50257), (40, 900)):
        x, t = _logits(n, v, "bf16", 19), _targets(n, v, 20)
        g = torch.ones(n, device=DEV)

        def step():
            r = ms.ops.token_logprobs(x, t, top=5, entropy=True)
            return [*r, ms.ops.token_logprobs_grad(x, t, r.lse, g, r.entropy, g)]

        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for seed in range(21, 25):
            x.copy_(_logits(n, v, "bf16", seed))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_refusals():
    x, t = _logits(4, 10, "fp32", 26), _targets(4, 10, 27)
    r = ms.ops.token_logprobs(x, t)
    g = torch.ones(4, device=DEV)
    with pytest.raises(ValueError, match="top"):
        ms.ops.token_logprobs(x, t, top=11)
    with pytest.raises(ValueError, match="top"):
        ms.ops.token_logprobs(x, t, top=-1)
    with pytest.raises(ValueError, match="top"):
        ms.ops.token_logprobs(_logits(2, 100, "fp32", 1), t[:2], top=65)
    with pytest.raises(ValueError, match="targets"):
        ms.ops.token_logprobs(x, t[:3])
    with pytest.raises(ValueError, match="targets"):
        ms.ops.token_logprobs(x, x)
    with pytest.raises(TypeError, match="targets"):
        ms.ops.token_logprobs(x, g)
    with pytest.raises(TypeError, match="logits"):
        ms.ops.token_logprobs(x.double(), t)
    with pytest.raises(ValueError, match="vocabulary"):
        ms.ops.token_logprobs(x[:, :0], t)
    with pytest.raises(RuntimeError, match="cpu"):
        ms.ops.token_logprobs(x.cpu(), t)
    with pytest.raises(RuntimeError, match="cpu"):
        ms.ops.token_logprobs(x, t.cpu())
    with pytest.raises(ValueError, match="lse"):
        ms.ops.token_logprobs_grad(x, t, r.lse[:2], g)
    with pytest.raises(TypeError, match="grad_logprob"):
        ms.ops.token_logprobs_grad(x, t, r.lse, g.double())
    with pytest.raises(ValueError, match="entropy"):
        ms.ops.token_logprobs_grad(x, t, r.lse, g, grad_entropy=g)
    with pytest.raises(RuntimeError, match="cpu"):
        ms.ops.token_logprobs_grad(x, t, r.lse.cpu(), g)
