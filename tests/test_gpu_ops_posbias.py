"""Relative position bias and its table's gradient against plain loops over buckets.

The bias is copied, so it is compared bit for bit.  A gradient is an fp32 sum of n values
and one rounding: n 2^-24 of the sum of magnitudes, half an ulp of the result."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch
import torch.nn.functional as F

import minispeed_amd as ms
from minispeed_amd import build
from tests import ops_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def side_bucket(away, n, distance):
    """By whole numbers alone."""
    one = n // 2
    if away < one:
        return away
    steps, s = n - one, 0
    while s + 1 < steps and away ** steps * one ** (s + 1) >= distance ** (s + 1) * one ** steps:
        s += 1
    return one + s


def bucket_map(queries, keys, first, buckets, distance, causal):
    """[queries, keys] of buckets; -1 where a key is out of reach."""
    n = buckets if causal else buckets // 2
    rels = range(-(first + queries - 1), keys - first)
    side = {}

    def of(rel):
        if rel > 0 and causal:
            return -1
        away = min(abs(rel), max(distance, n))
        if away not in side:
            side[away] = side_bucket(away, n, distance)
        return side[away] + (n if rel > 0 else 0)

    line = torch.tensor([of(r) for r in rels])
    at = torch.arange(keys)[None, :] - torch.arange(queries)[:, None] + queries - 1
    return line[at]


def check(heads, queries, keys, buckets, distance, causal, dtype, first=None, batch=(2,), seed=0):
    g = torch.Generator().manual_seed(seed)
    dt = ref.DTYPES[dtype]
    table = torch.randn(buckets, heads, generator=g).to(dt)
    at = bucket_map(queries, keys, keys - queries if first is None else first, buckets, distance, causal)
    got = ms.ops.position_bias(table.to(DEV), queries, keys, first=first, max_distance=distance,
                               causal=causal)
    want = torch.where((at < 0)[None], torch.tensor(-math.inf, dtype=dt),
                       table[at.clamp(min=0)].permute(2, 0, 1))
    assert got.shape == (heads, queries, keys) and got.dtype == dt
    assert torch.equal(got.cpu(), want)
    grad = torch.randn(*batch, heads, queries, keys, generator=g).to(dt)
    if causal:
        grad[..., at < 0] = math.nan           # (not looked at)
    dt_ = ms.ops.position_bias_grad(grad.to(DEV), buckets, first=first, max_distance=distance, causal=causal)
    flat = grad.double().reshape(-1, heads, queries * keys)
    total, size = (torch.zeros(buckets, heads, dtype=torch.float64) for _ in range(2))
    keep = at.reshape(-1) >= 0
    for part in flat:
        total.index_add_(0, at.reshape(-1)[keep], part[:, keep].T)
        size.index_add_(0, at.reshape(-1)[keep], part[:, keep].T.abs())
    count = torch.bincount(at.reshape(-1)[keep], minlength=buckets)[:, None] * len(flat)
    ref.close(dt_, total, size * (count + 2) * 2.0 ** -24 + ref.rounding(total, dt))
    return table.to(DEV), grad.to(DEV), dt_


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("queries,keys", [(1, 1), (1, 7), (2, 2), (5, 5), (1, 300), (33, 33), (64, 129),
                                          (130, 130), (3, 2100), (70, 4099), (300, 1025)])
def test_sizes(dtype, causal, queries, keys):
    check(3, queries, keys, 32, 128, causal, dtype, seed=queries + keys)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("buckets,distance", [(4, 2), (4, 3), (8, 128), (32, 9), (64, 257), (128, 65),
                                              (512, 512), (512, 5000), (6, 50), (32, 2 ** 31 - 1)])
def test_buckets(causal, buckets, distance):
    if causal:
        distance = max(distance, buckets // 2 + 1)
    check(2, 150, 700, buckets, distance, causal, "fp32", seed=buckets)
    if causal:
        check(2, 20, 90, buckets - 1, distance, causal, "bf16", seed=buckets)


@pytest.mark.parametrize("first", [0, 5, -40, 100, 5000, -5000])
def test_positions_of_the_queries(first):
    for causal in (False, True):
        check(2, 30, 50, 32, 64, causal, "fp16", first=first, seed=1)


def test_borders_of_the_buckets():
    """Distances on both sides of every border, some of them whole powers."""
    for buckets, distance in ((32, 128), (64, 2048), (16, 64), (36, 9 * 3 ** 9)):
        check(1, 1, 20000, buckets, distance, True, "fp32", batch=(1,))
        check(1, 3, 5000, buckets, distance, False, "fp32", first=2500, batch=())


def test_layouts():
    table, grad, want = check(6, 40, 72, 32, 64, False, "bf16", batch=(3, 2), seed=2)
    call = lambda g: ms.ops.position_bias_grad(g, 32, max_distance=64)  # noqa: E731
    wide = torch.zeros(3, 2, 6, 40, 75, dtype=grad.dtype, device=DEV)
    wide[..., 1:73] = grad
    assert torch.equal(call(wide[..., 1:73]), want)
    assert torch.equal(call(grad.transpose(0, 1).contiguous().transpose(0, 1)), want)
    assert torch.equal(call(grad.transpose(-1, -2).contiguous().transpose(-1, -2)), want)
    assert torch.equal(call(grad.permute(2, 0, 1, 3, 4).contiguous().permute(1, 2, 0, 3, 4)), want)
    one = grad[:1, :1]
    assert torch.equal(call(one.expand(3, 2, 6, 40, 72)), call(one.expand(3, 2, 6, 40, 72).contiguous()))
    assert torch.equal(call(torch.ones((), device=DEV).expand(6, 40, 72)), call(torch.ones(6, 40, 72, device=DEV)))
    bias = ms.ops.position_bias(table, 40, 72, max_distance=64)
    for t in (table.t().contiguous().t(), torch.stack([table, table], 2)[:, :, 0]):
        assert torch.equal(ms.ops.position_bias(t, 40, 72, max_distance=64), bias)


def test_nothing_to_do():
    table = torch.randn(32, 4, device=DEV)
    for heads, q, k in ((4, 0, 5), (4, 5, 0), (0, 5, 5)):
        assert ms.ops.position_bias(table[:, :heads], q, k).shape == (heads, q, k)
        g = ms.ops.position_bias_grad(torch.zeros(2, heads, q, k, device=DEV), 32)
        assert torch.equal(g, torch.zeros(32, heads, device=DEV))
    g = ms.ops.position_bias_grad(torch.zeros(0, 4, 5, 5, device=DEV), 32)
    assert torch.equal(g, torch.zeros(32, 4, device=DEV))


def test_rows_past_32_bits():
    table = torch.randn(32, 9, device=DEV).half()
    bias = ms.ops.position_bias(table, 16000, 16001, causal=True)      # 2.3e9 values
    for h, i in ((8, 15999), (8, 0), (4, 7000)):
        line = ms.ops.position_bias(table, 1, 16001, first=1 + i, causal=True)
        assert torch.equal(bias[h, i], line[h, 0])
    bias.fill_(2.0 ** -10)
    g = ms.ops.position_bias_grad(bias, 32, causal=True)
    # bucket 0: the pairs of distance 0, one for each query
    want = torch.full((9,), 16000 * 2.0 ** -10, device=DEV).half()
    assert torch.equal(g[0], want) and torch.equal(g[:, 0], g[:, 8])


def test_the_same_bits_every_time_and_on_another_stream():
    grad = torch.randn(4, 8, 500, 501, device=DEV).half()
    first = ms.ops.position_bias_grad(grad, 32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(side):
            again = ms.ops.position_bias_grad(grad, 32)
        side.synchronize()
        assert torch.equal(first, again)


def test_in_attention():
    """The mask of an attention whose gradient comes back to the table, against the table's own
    lookups in 64 bits and central differences."""
    torch.manual_seed(3)
    b, h, t, d = 2, 3, 37, 16
    q, k, v = (torch.randn(b, h, t, d, device=DEV) for _ in range(3))
    table = (torch.randn(16, h, device=DEV) * 0.5).requires_grad_()
    w = torch.randn(b, h, t, d, device=DEV)
    at = bucket_map(t, t, 0, 16, 20, True).to(DEV)

    def attend(table_, bias):
        s = (q.double() @ k.double().transpose(-1, -2).contiguous()) / math.sqrt(d) + bias
        return (torch.softmax(s, -1) @ v.double() * w.double()).sum()

    bias = ms.ops.position_bias(table, t, t, max_distance=20, causal=True)
    attend(table, bias.double()).backward()
    plain = table.detach().double().requires_grad_()

    def lookup(x):
        return x[at.clamp(min=0)].permute(2, 0, 1).masked_fill(at < 0, -math.inf)

    want, = torch.autograd.grad(attend(plain, lookup(plain)), plain)
    # (the bias's gradient is rounded to fp32 before it is summed over 2 x 37 x 37 values)
    assert float((table.grad.double() - want).abs().max()) <= 1e-5 * float(want.abs().max())
    step, direction = 1e-5, torch.randn(16, h, device=DEV).double()
    with torch.no_grad():
        up, down = (attend(None, lookup(plain + s * step * direction)) for s in (1, -1))
    slope = float(up - down) / (2 * step)
    parts = table.grad.double() * direction
    assert abs(slope - float(parts.sum())) <= 1e-5 * float(parts.abs().sum()) + 1e-6


def test_in_a_graph():
    table = torch.randn(32, 4, device=DEV).half()
    grad = torch.randn(2, 4, 100, 130, device=DEV).half()

    def step():
        return (ms.ops.position_bias(table, 100, 130, causal=True),
                ms.ops.position_bias_grad(grad, 32, causal=True))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(4):
        table.copy_(torch.randn(32, 4, device=DEV))
        grad.copy_(torch.randn(2, 4, 100, 130, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_refusals():
    table = torch.randn(32, 4, device=DEV)
    call, grad = ms.ops.position_bias, ms.ops.position_bias_grad
    for bad, causal in ((3, False), (2, False), (5, False), (514, False), (1, True), (513, True)):
        with pytest.raises(ValueError, match="buckets"):
            call(torch.zeros(bad, 4, device=DEV), 5, 5, max_distance=1000, causal=causal)
        with pytest.raises(ValueError, match="buckets"):
            grad(torch.zeros(4, 5, 5, device=DEV), bad, max_distance=1000, causal=causal)
    with pytest.raises(ValueError, match="max_distance"):
        call(table, 5, 5, max_distance=8)
    with pytest.raises(ValueError, match="max_distance"):
        call(table, 5, 5, max_distance=16, causal=True)
    with pytest.raises(ValueError, match="first"):
        call(table, 5, 5, first=2 ** 41)
    with pytest.raises(ValueError, match="queries"):
        call(table, -1, 5)
    with pytest.raises(ValueError, match="table"):
        call(table[0], 5, 5)
    with pytest.raises(TypeError, match="table"):
        call(table.double(), 5, 5)
    with pytest.raises(ValueError, match="grad"):
        grad(table, 32)
    with pytest.raises(ValueError, match="grad"):
        grad(table, 32, first=0)


def test_the_library_by_itself():
    lib = ctypes.CDLL(build.OPS_OUTPUT)
    P, I32, I64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64
    lib.ms_position_bias_grad_workspace.restype = I64
    grad = torch.randn(3, 4, 50, 60, device=DEV)
    need = lib.ms_position_bias_grad_workspace(I32(0), I64(32), I64(3), I64(4), I64(50), I64(60))
    work = torch.full((need + 4096,), 77, dtype=torch.uint8, device=DEV)
    out = torch.empty(32, 4, device=DEV)
    assert lib.ms_position_bias_grad(P(grad.data_ptr()), I32(0), I64(3), I64(12000), I64(4), I64(3000),
                                     I64(50), I64(60), I64(60), I64(10), I64(32), I64(128), I32(0),
                                     P(out.data_ptr()), P(work.data_ptr()), I64(need),
                                     P(torch.cuda.current_stream().cuda_stream)) == 0
    assert bool((work[need:] == 77).all())
    assert torch.equal(out, ms.ops.position_bias_grad(grad, 32))
