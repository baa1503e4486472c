"""Log probabilities without logits, and their gradients, against 64-bit sums.

Tolerances.  With u = 2^-24, a logit of K products is an fp32 sum of exact products
(2-byte operands), whose order is the kernel's: K u of the sum of magnitudes, twice for
sums that drop bits instead of rounding them; three planes of a 32-bit operand leave out
products below 2^-22 of the magnitudes.  With L the largest such error of a row's logits:
a term exp(x - base) is off by L + 2^-22 (|x| + |base| + 1) relative (argument and
exponential), the sum of V terms, up to 128 + V / 128 of them one after the other, by as
many u more, and lse by that and 2^-22 |lse|.
Gradients: each term d W is off by what its p is, by half an ulp of d (2^-24 of three
planes), by (terms) u in the sums; the result is rounded once.  In fp16, rows of d are scaled so
that half a subnormal step (2^-25) is 2^-38 of the larger of a row's two terms (scaled to 2^13 or more); hidden, multiplied by a power of
two up to the ratio of the rows' bounds, is off by 2^-25 of the largest row's scale.
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
U = 2.0 ** -24


def make(n, d, v, dtype, seed, std=0.3, ignored=0.2):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = ref.DTYPES[dtype]
    h = torch.randn(n, d, generator=g, device=DEV).to(dt)
    w = (torch.randn(v, d, generator=g, device=DEV) * (std if d < 64 else std * 8 / d ** 0.5)).to(dt)
    t = torch.randint(0, v, (n,), generator=g, device=DEV)
    t[torch.rand(n, generator=g, device=DEV) < ignored] = -100
    gr = torch.randn(n, generator=g, device=DEV) / n
    gl = torch.randn(n, generator=g, device=DEV) * 0.1 / n
    return h, w, t, gr, gl


def _flat(h, w):
    return h.reshape(-1, h.shape[-1]).double(), w.double()


def forward(h, w, t, scale=1.0, ignore=-100):
    """(logprob, lse, tolerances of both, logits) in 64 bits."""
    hd, wd = _flat(h, w)
    t = t.reshape(-1).long()
    n, k, v = len(hd), hd.shape[1], len(wd)
    x = hd @ wd.T * scale
    size = (hd.abs() @ wd.abs().T * abs(scale)).amax(1)
    lse = torch.logsumexp(x, 1)
    picked = x.gather(1, t.clamp(0, v - 1)[:, None])[:, 0]
    logprob = torch.where(t == ignore, 0.0, picked - lse)
    logprob = torch.where((t != ignore) & ((t < 0) | (t >= v)), NAN, logprob)
    part = 2.0 ** -22 if h.dtype == torch.float32 else 0.0
    big = (x.abs().amax(1) + lse.abs() + 1) * 2.0 ** -22
    logit = size * (2 * k * U * (6 if part else 1) + 4 * part)
    tol = logit + 2 * big + (128 + v / 128) * U
    return logprob, lse, tol + logit + big, tol, x


def backward(h, w, t, gr, gl, scale=1.0, ignore=-100):
    hd, wd = _flat(h, w)
    t = t.reshape(-1).long()
    n, k, v = len(hd), hd.shape[1], len(wd)
    _, lse, tol_p, tol_l, x = forward(h, w, t, scale, ignore)
    g = torch.where(t == ignore, 0.0, gr.reshape(-1).double()) if gr is not None else torch.zeros(n, device=DEV).double()
    l = gl.reshape(-1).double() if gl is not None else torch.zeros_like(g)
    p = torch.exp(x - lse[:, None])
    at = t.clamp(0, v - 1)[:, None]
    d = p * (l - g)[:, None]
    size = d.abs()
    d.scatter_add_(1, at, g[:, None])
    size.scatter_add_(1, at, g.abs()[:, None])
    dh, dw = scale * d @ wd, scale * d.T @ hd
    half = {torch.float32: 2.0 ** -22, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[h.dtype]
    rel = half + (tol_p + tol_l)[:, None] + 2.0 ** -21
    many = 2 * U * (6 if h.dtype == torch.float32 else 1)
    bound = (l - g).abs() + g.abs()
    # The exponential instruction gives 0 in the place of numbers below 2^-126, the smallest
    # normal one, so p is off by that; d and its planes by as much where they are so small.
    small = bound * 2.0 ** -38 if h.dtype == torch.float16 else (bound + 4) * 2.0 ** -126
    err = size * rel + small[:, None]
    th = abs(scale) * (err + size * many * v) @ wd.abs() + ref.rounding(dh, h.dtype)
    tw = abs(scale) * (err + size * many * n).T @ hd.abs() + ref.rounding(dw, h.dtype)
    if h.dtype == torch.float16 and n:
        tw = tw + abs(scale) * (2.0 ** -24 * size * (bound.max() / bound.clamp(min=1e-300))[:, None]).sum(0)[:, None]
    return dh, dw, th, tw


def check(h, w, t, gr, gl, scale=1.0, ignore=-100):
    r = ms.ops.linear_logprobs(h, w, t, scale=scale, ignore_index=ignore)
    assert r.logprob.shape == r.lse.shape == t.shape and r.lse.dtype == r.logprob.dtype == torch.float32
    logprob, lse, tol_p, tol_l, _ = forward(h, w, t, scale, ignore)
    what = f"{tuple(h.shape)} {tuple(w.shape)} {h.dtype}"
    ref.close(r.lse.reshape(-1), lse, tol_l, "lse " + what)
    ref.close(r.logprob.reshape(-1), logprob, tol_p, "logprob " + what)
    dh, dw = ms.ops.linear_logprobs_grad(h, w, t, r.lse, gr, gl, scale=scale, ignore_index=ignore)
    assert dh.shape == h.shape and dw.shape == w.shape and dh.dtype == dw.dtype == h.dtype
    eh, ew, th, tw = backward(h, w, t, gr, gl, scale, ignore)
    ref.close(dh.reshape(eh.shape), eh, th, "dhidden " + what)
    ref.close(dw, ew, tw, "dweight " + what)
    return r, dh, dw


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("n,d,v", [(1, 1, 1), (1, 64, 129), (3, 7, 65), (31, 64, 128), (33, 72, 300),
                                   (64, 8, 1000), (65, 65, 257), (127, 200, 513), (130, 63, 4097),
                                   (300, 136, 1001), (1000, 24, 70)])
def test_sizes(dtype, n, d, v):
    check(*make(n, d, v, dtype, n + d + v))


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("n,d,v", [(2100, 72, 8200), (70, 4096, 4100), (4200, 4096, 70)])
def test_wide_tiles(dtype, n, d, v):
    """Each of the products by the largest tiles, with edges inside them."""
    check(*make(n, d, v, dtype, n + d))


@pytest.mark.parametrize("n,d,v", [(700, 257, 3001), (390, 65, 22000), (500, 131, 9001), (385, 2056, 700)])
def test_many_tokens_of_32_bits(n, d, v):
    """Those are multiplied by planes of 16 bits."""
    h, w, t, gr, gl = make(n, d, v, "fp32", n)
    first = check(h, w, t, gr, gl)
    base = torch.zeros(v, d + 3, device=DEV)
    base[:, 1:d + 1] = w
    again = check(h, base[:, 1:d + 1], t.int(), gr, gl, scale=1.0)
    assert all(torch.equal(a, b) for a, b in zip((*first[0], *first[1:]), (*again[0], *again[1:])))
    check(h * 1e-3, w * 1e3, t, gr, None, scale=-0.5)
    bad = h.clone()
    bad[3, 1], bad[4, 0] = NAN, INF
    r = ms.ops.linear_logprobs(bad, w, t)
    assert r.lse[3].isnan() and r.lse[4].isnan()
    keep = torch.ones(n, dtype=torch.bool, device=DEV)
    keep[3:5] = False
    assert torch.equal(r.lse[keep], first[0].lse[keep])


@pytest.mark.parametrize("n,d,v", [(384, 520, 3001), (383, 65, 22001), (300, 2050, 701)])
def test_tokens_of_32_bits_as_they_are(n, d, v):
    check(*make(n, d, v, "fp32", n))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_several_pieces_of_the_vocabulary(dtype):
    check(*make(60000, 16, 3000, dtype, 5))


def test_few_tokens_of_a_wide_head():
    check(*make(4, 1024, 30011, "bf16", 6))
    check(*make(1, 4096, 5003, "fp16", 7))


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_layouts(dtype):
    n, d, v = 90, 72, 333
    h, w, t, gr, gl = make(n, d, v, dtype, 8)
    first = check(h, w, t, gr, gl)
    same = lambda r: all(torch.equal(a.reshape(b.shape), b) for a, b in zip((*r[0], *r[1:]), (*first[0], *first[1:])))  # noqa: E731
    base = torch.zeros(n, d + 9, dtype=h.dtype, device=DEV)
    base[:, 3:3 + d] = h
    assert same(check(base[:, 3:3 + d], w, t, gr, gl))                    # rows off 16 bytes
    base = torch.zeros(v, d + 8, dtype=h.dtype, device=DEV)
    base[:, 8:] = w
    assert same(check(h, base[:, 8:], t, gr, gl))                         # rows apart
    assert same(check(h, w.t().contiguous().t(), t.int(), gr, gl))        # columns first, 4-byte ids
    assert same(check(h.view(9, 10, d).transpose(0, 1).contiguous().transpose(0, 1),
                      w, t.view(9, 10), gr.view(9, 10), gl.view(9, 10)))
    assert same(check(h, w, torch.stack([t, t], 1)[:, 0], torch.stack([gr, gr], 1)[:, 1], gl))


@pytest.mark.parametrize("scale", [0.125, -1.5, 0.0, 8.0])
def test_scale(scale):
    for dtype in ("fp32", "fp16", "bf16"):
        check(*make(70, 40, 200, dtype, 9), scale=scale)


def test_gradients_alone_and_none():
    h, w, t, gr, gl = make(40, 64, 300, "bf16", 10)
    check(h, w, t, gr, None)
    check(h, w, t, None, gl)
    r = ms.ops.linear_logprobs(h, w, t)
    dh, dw = ms.ops.linear_logprobs_grad(h, w, t, r.lse, None)
    assert not dh.any() and not dw.any()
    for need in ((True, False), (False, True)):
        a, b = h.clone().requires_grad_(need[0]), w.clone().requires_grad_(need[1])
        (ms.ops.linear_logprobs(a, b, t).logprob * gr).sum().backward()
        one, two = ms.ops.linear_logprobs_grad(h, w, t, r.lse, gr)
        assert (a.grad is None) != need[0] and (b.grad is None) != need[1]
        assert torch.equal(a.grad if need[0] else b.grad, one if need[0] else two)


def test_no_tokens():
    for dtype in ("fp32", "fp16"):
        h, w, t, gr, gl = make(0, 33, 20, dtype, 11)
        r = ms.ops.linear_logprobs(h, w, t)
        assert r.lse.shape == (0,)
        dh, dw = ms.ops.linear_logprobs_grad(h, w, t, r.lse, gr)
        assert dh.shape == (0, 33) and torch.equal(dw, torch.zeros_like(w))


def test_targets_outside_the_vocabulary():
    h, w, t, gr, gl = make(40, 16, 100, "fp32", 12, ignored=0.0)
    t[3], t[4], t[5] = 100, -1, -100
    r = ms.ops.linear_logprobs(h, w, t)
    assert r.logprob[3].isnan() and r.logprob[4].isnan() and r.logprob[5] == 0
    assert torch.isfinite(r.lse).all()
    dh, _ = ms.ops.linear_logprobs_grad(h, w, t, r.lse, gr, gl)
    bad = dh.isnan().any(1)
    assert bad.nonzero()[:, 0].tolist() == [3, 4]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_gradients_of_very_different_rows(dtype):
    """Row gradients over many powers of two: each row of dhidden keeps its own precision."""
    h, w, t, gr, gl = make(200, 64, 500, dtype, 13, ignored=0.0)
    gr = gr.abs() * 2.0 ** torch.arange(200, device=DEV).remainder(12)
    check(h, w, t, gr, None)
    check(h, w, t, gr * 1e-6, None)
    tiny = gr.clone()
    tiny[::2] *= 1e-12
    r = ms.ops.linear_logprobs(h, w, t)
    dh, _ = ms.ops.linear_logprobs_grad(h, w, t, r.lse, tiny * 1e4)
    eh, _, th, _ = backward(h, w, t, tiny * 1e4, None)
    if dtype == "fp16":
        # from 65520 on (half a step above the largest number) the rounding gives infinity;
        # what is that within its tolerance may be either
        edge = (eh.abs() - 65520.0).abs() <= th
        eh = torch.where(eh.abs() >= 65520.0, torch.sign(eh) * INF, eh)
        dh, eh = dh.double().masked_fill(edge, 0.0), eh.masked_fill(edge, 0.0)
    ref.close(dh, eh, th)


def test_many_rows_of_very_different_gradients():
    """fp16 beyond the rows that one block numbers; gradients up to the largest."""
    h, w, t, gr, gl = make(20000, 16, 70, "fp16", 30, ignored=0.0)
    check(h, w, t, gr * 2.0 ** torch.arange(20000, device=DEV).remainder(9), gl)
    h, w, t, gr, gl = make(40, 16, 70, "fp16", 31, ignored=0.0)
    huge = torch.full_like(gr, 2.0 ** 127)
    r = ms.ops.linear_logprobs(h, w, t, scale=2.0 ** -125)
    dh, dw = ms.ops.linear_logprobs_grad(h, w, t, r.lse, huge, scale=2.0 ** -125)
    eh, ew, th, tw = backward(h, w, t, huge, None, 2.0 ** -125)
    ref.close(dh, eh, th)
    ref.close(dw, ew, tw)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_infinities_and_nan(dtype):
    h, w, t, gr, gl = make(70, 32, 300, dtype, 14, ignored=0.0)
    w[:, 0] = w[:, 0].abs() + 0.25
    good = ms.ops.linear_logprobs(h, w, t)
    h2 = h.clone()
    h2[5, 3], h2[6, 0] = NAN, INF
    r = ms.ops.linear_logprobs(h2, w, t)
    assert r.lse[5].isnan() and r.lse[6].isnan() and r.logprob[5].isnan() and r.logprob[6].isnan()
    keep = torch.ones(70, dtype=torch.bool, device=DEV)
    keep[5:7] = False
    assert torch.equal(r.lse[keep], good.lse[keep]) and torch.equal(r.logprob[keep], good.logprob[keep])
    dh, _ = ms.ops.linear_logprobs_grad(h2, w, t, r.lse, gr)
    eh, _ = ms.ops.linear_logprobs_grad(h, w, t, good.lse, gr)
    assert dh[5].isnan().all() and dh[6].isnan().all() and torch.equal(dh[keep], eh[keep])


def test_a_row_without_a_finite_logit():
    """Only -inf: lse is -inf, and the row has no gradient."""
    for dtype in ("fp16", "bf16"):
        h, w, t, gr, gl = make(40, 32, 300, dtype, 15, ignored=0.0)
        w[:, 0] = w[:, 0].abs() + 0.25
        h[7] = 0.0
        h[7, 0] = -INF
        r = ms.ops.linear_logprobs(h, w, t)
        assert r.lse[7] == -INF and r.logprob[7] == -INF
        dh, _ = ms.ops.linear_logprobs_grad(h, w, t, r.lse, gr, gl)
        assert not dh[7].any() and torch.isfinite(dh).all()


def test_logits_far_from_zero():
    """Hidden states of large norm: logits of some hundreds, one far above the others."""
    for dtype in ("fp32", "bf16"):
        h, w, t, gr, gl = make(66, 64, 700, dtype, 16)
        check(h * 100, w, t, gr, gl)
        check(h * -100, w.abs(), t, gr, gl)


def test_rows_past_32_bits():
    """A weight of more than 2^31 elements, its last rows among the targets."""
    d, v = 65536, 33000
    w = torch.zeros(v, d, device=DEV, dtype=torch.bfloat16)
    w[-5:] = torch.randn(5, d, device=DEV) * 0.01
    h = torch.randn(3, d, device=DEV).bfloat16()
    t = torch.tensor([v - 1, v - 3, 0], device=DEV)
    r = ms.ops.linear_logprobs(h, w, t)
    x = torch.zeros(3, v, device=DEV, dtype=torch.float64)
    x[:, -5:] = h.double() @ w[-5:].double().T
    lse = torch.logsumexp(x, 1)
    ref.close(r.lse, lse, 1e-4 * torch.ones(3))
    ref.close(r.logprob, x.gather(1, t[:, None])[:, 0] - lse, 1e-4 * torch.ones(3))
    g = torch.tensor([1.0, -2.0, 0.5], device=DEV)
    _, dw = ms.ops.linear_logprobs_grad(h, w, t, r.lse, g)
    dd = -torch.exp(x - lse[:, None]) * g.double()[:, None]
    dd.scatter_add_(1, t[:, None], g.double()[:, None])
    for rows in (slice(0, 4), slice(v - 8, v)):
        want = dd[:, rows].T @ h.double()
        size = dd[:, rows].abs().T @ h.double().abs()
        # as in backward(), with logits off by 2 d u |h||w| ~ 2e-4 at most
        ref.close(dw[rows], want, size * (2.0 ** -8 + 1e-3) + ref.rounding(want, torch.bfloat16))


def test_the_same_bits_every_time_and_on_another_stream():
    for dtype in ("fp16", "fp32"):
        h, w, t, gr, gl = make(3000, 72, 5000, dtype, 17)
        r = ms.ops.linear_logprobs(h, w, t)
        grads = ms.ops.linear_logprobs_grad(h, w, t, r.lse, gr, gl)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        for _ in range(3):
            with torch.cuda.stream(side):
                again = ms.ops.linear_logprobs(h, w, t)
                more = ms.ops.linear_logprobs_grad(h, w, t, again.lse, gr, gl)
            side.synchronize()
            assert all(torch.equal(a, b) for a, b in zip((*r, *grads), (*again, *more)))


def test_autograd_against_the_formula_and_differences():
    h, w, t, _, _ = make(6, 20, 101, "fp32", 18)
    h.requires_grad_(), w.requires_grad_()
    r = ms.ops.linear_logprobs(h, w, t, scale=0.7)
    (r.logprob.sum() * -0.5 + 0.01 * (r.lse ** 2).sum()).backward()
    gr, gl = torch.full((6,), -0.5, device=DEV), (0.02 * r.lse).detach()
    eh, ew, th, tw = backward(h.detach(), w.detach(), t, gr, gl, 0.7)
    ref.close(h.grad, eh, th)
    ref.close(w.grad, ew, tw)

    def loss(a, b):
        lp, lse, _, _, _ = forward(a, b, t, 0.7)
        return float(lp.sum() * -0.5 + 0.01 * (lse ** 2).sum())

    # central differences of the 64-bit loss: step^2 of third derivatives of order 10, 2^-50 / step
    g = torch.Generator(device=DEV).manual_seed(19)
    step = 1e-5
    for x, grad, k in ((h, h.grad, 0), (w, w.grad, 1)):
        v = torch.randn(x.shape, generator=g, device=DEV).double()
        at = [h.detach().double(), w.detach().double()]
        up, down = list(at), list(at)
        up[k], down[k] = at[k] + step * v, at[k] - step * v
        slope = (loss(*up) - loss(*down)) / (2 * step)
        parts = grad.double() * v
        assert abs(slope - float(parts.sum())) <= 1e-5 * float(parts.abs().sum()) + 1e-7


def test_in_a_graph():
    for n, d, v, dtype in ((3, 64, 1000, "bf16"), (200, 70, 900, "fp16"), (100, 32, 300, "fp32")):
        h, w, t, gr, gl = make(n, d, v, dtype, 20)

        def step():
            r = ms.ops.linear_logprobs(h, w, t)
            return [*r, *ms.ops.linear_logprobs_grad(h, w, t, r.lse, gr, gl)]

        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for seed in range(21, 25):
            h.copy_(make(n, d, v, dtype, seed)[0])
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_refusals():
    h, w, t, gr, _ = make(4, 8, 10, "fp32", 26)
    r = ms.ops.linear_logprobs(h, w, t)
    call = ms.ops.linear_logprobs
    with pytest.raises(ValueError, match="weight"):
        call(h, w[:, :7], t)
    with pytest.raises(ValueError, match="weight"):
        call(h, w[0], t)
    with pytest.raises(TypeError, match="dtype"):
        call(h, w.half(), t)
    with pytest.raises(TypeError, match="hidden"):
        call(h.double(), w.double(), t)
    with pytest.raises(ValueError, match="vocabulary"):
        call(h, w[:0], t)
    with pytest.raises(ValueError, match="width"):
        call(h[:, :0], w[:, :0], t)
    with pytest.raises(ValueError, match="targets"):
        call(h, w, t[:3])
    with pytest.raises(TypeError, match="targets"):
        call(h, w, gr)
    with pytest.raises(RuntimeError, match="cpu"):
        call(h, w.cpu(), t)
    with pytest.raises(RuntimeError, match="cpu"):
        call(h, w, t.cpu())
    grad = ms.ops.linear_logprobs_grad
    with pytest.raises(ValueError, match="lse"):
        grad(h, w, t, r.lse[:2], gr)
    with pytest.raises(TypeError, match="grad_logprob"):
        grad(h, w, t, r.lse, gr.double())
    with pytest.raises(RuntimeError, match="cpu"):
        grad(h, w, t, r.lse, gr, gr.cpu())


def test_the_library_by_itself():
    """The C entries with a workspace of exactly the size that they ask for."""
    lib = ctypes.CDLL(build.OPS_OUTPUT)
    P, I64, F = ctypes.c_void_p, ctypes.c_int64, ctypes.c_float
    lib.ms_linear_logprobs_workspace.restype = lib.ms_linear_logprobs_grad_workspace.restype = I64
    n, d, v = 70, 40, 300
    h, w, t, gr, gl = make(n, d, v, "bf16", 27)
    hr, wr = Rows(h.data_ptr(), n, d, n, 0, d, 2, 0), Rows(w.data_ptr(), v, d, v, 0, d, 2, 0)
    ids = Tokens(t.data_ptr(), n, n, 0, 1, 1, 0)
    ref_ = ctypes.byref
    stream = P(torch.cuda.current_stream().cuda_stream)
    need = lib.ms_linear_logprobs_workspace(ref_(hr), ref_(wr))
    more = lib.ms_linear_logprobs_grad_workspace(ref_(hr), ref_(wr))
    guard = 4096
    work = torch.full((max(need, more) + guard,), 77, dtype=torch.uint8, device=DEV)
    lp, lse = torch.empty(n, device=DEV), torch.empty(n, device=DEV)
    assert lib.ms_linear_logprobs(ref_(hr), ref_(wr), ref_(ids), F(1), I64(-100), P(lp.data_ptr()),
                                  P(lse.data_ptr()), P(work.data_ptr()), I64(need), stream) == 0
    assert bool((work[need:] == 77).all())
    work.fill_(77)
    dh, dw = torch.empty_like(h), torch.empty_like(w)
    assert lib.ms_linear_logprobs_grad(ref_(hr), ref_(wr), ref_(ids), F(1), I64(-100), P(lse.data_ptr()),
                                       P(gr.data_ptr()), P(gl.data_ptr()), P(dh.data_ptr()),
                                       P(dw.data_ptr()), P(work.data_ptr()), I64(more), stream) == 0
    assert bool((work[more:] == 77).all())
    r = ms.ops.linear_logprobs(h, w, t)
    eh, ew = ms.ops.linear_logprobs_grad(h, w, t, r.lse, gr, gl)
    assert torch.equal(lse, r.lse) and torch.equal(lp, r.logprob)
    assert torch.equal(dh, eh) and torch.equal(dw, ew)
