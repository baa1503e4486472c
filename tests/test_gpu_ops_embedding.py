"""The token embedding and its gradient against 64-bit sums.

Tolerances: the lookup is one fp32 product and one rounding, so it is compared
bit for bit.  A gradient row of n tokens is n - 1 fp32 additions, one fp32
product and one rounding: n 2^-24 of the sum of magnitudes and half a unit in
the last place of the result.
"""

from __future__ import annotations

import ctypes

import pytest
import torch

import minispeed_amd as ms
from minispeed_amd import build
from tests import ops_reference as ref
from tests.test_ops_abi import Rows, Tokens

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _rand(shape, dtype, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(ref.DTYPES[dtype]).to(DEV)


def _ids(n, rows, seed, kind="zipf"):
    g = torch.Generator().manual_seed(seed)
    if kind == "same":
        return torch.full((n,), rows // 2, device=DEV)
    if kind == "uniform":
        return torch.randint(0, rows, (n,), generator=g).to(DEV)
    if kind == "sorted":
        return torch.randint(0, rows, (n,), generator=g).sort().values.to(DEV)
    u = torch.rand(n, generator=g)
    rank = (torch.exp(u * torch.log(torch.tensor(float(rows)))) - 1).long().clamp(0, rows - 1)
    return ((rank * 7919) % rows).to(DEV)


def check_grad(grad, ids, rows, scale=1.0, padding_idx=None):
    got = ms.ops.embedding_grad(grad, ids, rows, scale=scale, padding_idx=padding_idx)
    assert got.shape == (rows, grad.shape[-1]) and got.dtype == grad.dtype
    want, size, count = ref.embedding_grad(grad, ids, rows, scale, padding_idx)
    tol = size * (count + 2) * 2.0 ** -24 + ref.rounding(want, grad.dtype)
    ref.close(got, want, tol, f"embedding_grad {tuple(grad.shape)} rows {rows}")
    assert torch.equal(got[(count[:, 0] == 0).to(DEV)],
                       torch.zeros(int((count == 0).sum()), grad.shape[-1], dtype=grad.dtype,
                                   device=DEV))
    return got


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("rows,width,n", [(512, 256, 1024), (7, 1, 5), (1, 64, 3), (300, 257, 1),
                                          (1000, 768, 4097), (50257, 100, 333), (513, 1024, 63),
                                          (129, 2050, 65)])
def test_lookup_is_the_rounded_product(dtype, rows, width, n):
    w, ids = _rand((rows, width), dtype, 1), _ids(n, rows, 2, "uniform")
    for scale in (1.0, width ** 0.5, -0.3):
        got = ms.ops.embedding(ids, w, scale=scale)
        want = (w[ids].float() * scale).to(w.dtype)
        assert got.shape == (n, width) and torch.equal(got, want)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_lookup_layouts(dtype):
    big = _rand((64, 200), dtype, 3)
    for w in (big[:, :96], big[:, 3:99], big[::2], big[5:, :96], big.t()[:64], big[:, ::2]):
        batch = _ids(8 * 33, w.shape[0], 4, "uniform").view(8, 33)
        for ids in (batch, batch[:, :-1], batch[:, 1:], batch.t(), batch.int()[:, :-1],
                    batch.view(2, 4, 33)[:, 1:, :-1], batch[:, :1], batch[3, 5], batch[:0],
                    batch[:1].expand(5, 33)):
            got = ms.ops.embedding(ids, w, scale=2.0)
            want = (w[ids.long()].float() * 2.0).to(w.dtype)
            assert got.shape == want.shape and torch.equal(got, want)


def test_lookup_outside_the_table_is_nan():
    w = _rand((10, 40), "fp16", 5)
    ids = torch.tensor([0, -1, 9, 10, 2 ** 40, -2 ** 62], device=DEV)
    got = ms.ops.embedding(ids, w)
    assert torch.equal(got[[0, 2]], w[[0, 9]])
    assert bool(torch.isnan(got[[1, 3, 4, 5]]).all())


def test_lookup_past_32_bits():
    rows, width = 40_000, 65_536                              # 2.6e9 values, 5.2 GB
    w = torch.zeros(rows, width, dtype=torch.bfloat16, device=DEV)
    w[-1] = 3.0
    w[rows // 2, -1] = 2.0
    got = ms.ops.embedding(torch.tensor([rows - 1, rows // 2, 0], device=DEV), w)
    assert bool((got[0] == 3.0).all()) and got[1, -1] == 2.0 and not bool(got[2].any())
    grad = ms.ops.embedding_grad(got, torch.tensor([rows - 1, 1, 1], device=DEV), rows)
    assert bool((grad[-1] == 3.0).all()) and grad[1, -1] == 2.0
    assert not bool(grad[2:-1].any())


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("kind", ["zipf", "uniform", "same", "sorted"])
@pytest.mark.parametrize("rows,width,n", [(512, 256, 1024), (3, 64, 700), (1, 8, 1), (1025, 100, 1),
                                          (2049, 136, 2500), (50257, 24, 9000), (70_001, 8, 33),
                                          (333, 1, 40), (100, 515, 257), (64, 1032, 65)])
def test_grad(dtype, kind, rows, width, n):
    check_grad(_rand((n, width), dtype, 7, 0.1), _ids(n, rows, 8, kind), rows, scale=1.5)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("kind", ["same", "zipf", "uniform"])
@pytest.mark.parametrize("width", [257, 513, 1025, 1344, 2050, 4099])
def test_grad_of_wide_rows(dtype, kind, width):
    """Rows that several blocks share; the last part of one may be a single column."""
    for rows, n in ((2, 1000), (77, 300), (700, 1024)):
        check_grad(_rand((n, width), dtype, 29, 0.1), _ids(n, rows, 30, kind), rows)
        dirty = torch.full((rows, width), float("nan"), dtype=ref.DTYPES[dtype], device=DEV)
        del dirty                                 # the allocator hands it out again
        assert not bool(torch.isnan(ms.ops.embedding_grad(
            torch.ones(3, width, dtype=ref.DTYPES[dtype], device=DEV),
            torch.tensor([0, 1, 1], device=DEV), rows)).any())


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("width", [4, 5, 255, 257, 259, 260, 513, 514, 515, 516, 1025, 1027, 1344, 2049,
                                   2050, 2051, 2052, 2305, 4099, 8193])
def test_grad_adds_every_column_in_the_same_order(dtype, width):
    """Few tokens, whose columns several blocks may share: gradients that are alike in
    all columns have sums that are, bit for bit, on every call."""
    for rows, n, kind in ((2, 1000, "same"), (700, 1024, "same"), (1500, 777, "zipf"),
                          (3000, 1000, "same"), (8000, 333, "same")):
        ids = _ids(n, rows, 31, kind)
        g = _rand((n, 1), dtype, 32).expand(n, width).contiguous()
        first = ms.ops.embedding_grad(g, ids, rows)
        assert torch.equal(first, first[:, :1].expand(rows, width))
        assert torch.equal(ms.ops.embedding_grad(g, ids, rows), first)


@pytest.mark.parametrize("kind", ["same", "zipf"])
def test_grad_of_many_tokens(kind):
    check_grad(_rand((70_000, 72), "bf16", 9, 0.1), _ids(70_000, 5000, 10, kind), 5000)


@pytest.mark.parametrize("rows,width,n", [(50257, 768, 100), (128256, 1024, 3000), (9001, 515, 2500),
                                          (400, 64, 30), (3, 40000, 2100), (70000, 1, 5000)])
def test_grad_writes_every_row(rows, width, n):
    for dtype in ("bf16", "fp32"):
        g, ids = _rand((n, width), dtype, 27), _ids(n, rows, 28)
        dirty = torch.full((rows, width), float("nan"), dtype=g.dtype, device=DEV)
        at = dirty.data_ptr()
        del dirty                                 # the allocator hands it out again
        got = ms.ops.embedding_grad(g, ids, rows)
        assert got.data_ptr() == at
        seen = torch.zeros(rows, dtype=torch.bool, device=DEV)
        seen[ids] = True
        assert not bool(got[~seen].any())
        want = torch.zeros(rows, width, device=DEV).index_add_(0, ids, g.float())
        assert torch.allclose(got.float(), want, rtol=0.01, atol=0.1)


def test_grad_of_no_tokens_is_zeros():
    got = ms.ops.embedding_grad(torch.empty(0, 48, device=DEV),
                                torch.empty(0, dtype=torch.int64, device=DEV), 100)
    assert got.shape == (100, 48) and not bool(got.any())
    assert ms.ops.embedding_grad(torch.empty(2, 0, device=DEV),
                                 torch.zeros(2, dtype=torch.int64, device=DEV), 3).shape == (3, 0)


def test_grad_layouts():
    rows, width = 90, 64
    big = _rand((6, 40, 200), "bf16", 11)
    batch = _ids(6 * 40, rows, 12).view(6, 40)
    for g, ids in ((big[:, :, :width], batch), (big[:, 1:, 3:3 + width], batch[:, :-1]),
                   (big[:, :, :width].transpose(0, 1), batch.t()),
                   (big[:, :, ::2][:, :, :width], batch.int()),
                   (big[:1, :, :width].expand(6, 40, width), batch),
                   (big[:, :, :1].expand(6, 40, width), batch)):
        check_grad(g, ids, rows)


def test_grad_leaves_padding_and_strangers_out():
    ids = torch.tensor([3, 5, -1, 5, 9, 10, 3, -2 ** 60, 2 ** 33 + 3, 5], device=DEV)
    g = _rand((10, 70), "fp32", 13)
    check_grad(g, ids, 10, padding_idx=5)
    check_grad(g, ids, 10)
    assert torch.equal(ms.ops.embedding_grad(g, ids, 10, padding_idx=-5),
                       ms.ops.embedding_grad(g, ids, 10, padding_idx=5))


def test_grad_passes_infinities_on():
    g = _rand((600, 40), "fp16", 14)
    ids = _ids(600, 20, 15)
    g[17, 3], g[18, 4] = float("inf"), float("nan")
    got = ms.ops.embedding_grad(g, ids, 20)
    assert torch.isinf(got[ids[17], 3]) and torch.isnan(got[ids[18], 4])
    rest = torch.ones_like(got, dtype=torch.bool)
    rest[ids[17], 3] = rest[ids[18], 4] = False
    assert bool(torch.isfinite(got[rest]).all())


def test_grad_is_the_same_bits_every_time_and_at_any_alignment():
    n, rows, width = 5000, 700, 264
    ids = _ids(n, rows, 16)
    g = _rand((n, width), "bf16", 17)
    first = ms.ops.embedding_grad(g, ids, rows)
    shifted = torch.empty(n * width + 1, dtype=g.dtype, device=DEV)[1:].view(n, width).copy_(g)
    wide = torch.empty(n, width + 3, dtype=g.dtype, device=DEV)[:, 3:].copy_(g)
    for other in (g, shifted, wide):
        for _ in range(3):
            assert torch.equal(ms.ops.embedding_grad(other, ids.int(), rows), first)


def test_autograd_and_another_stream():
    rows, width = 211, 96
    w = _rand((rows, width), "fp32", 18).requires_grad_()
    ids = _ids(300, rows, 19).view(4, 75)
    up = _rand((4, 75, width), "fp32", 20)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ms.ops.embedding(ids, w, scale=3.0, padding_idx=int(ids[0, 0])).backward(up)
    torch.cuda.current_stream().wait_stream(side)
    want, size, count = ref.embedding_grad(up, ids, rows, 3.0, int(ids[0, 0]))
    ref.close(w.grad, want, size * (count + 2) * 2.0 ** -24 + ref.rounding(want, torch.float32))
    # against differences: the loss is linear in the table, so any step is exact
    # up to rounding; steps of 2^-3 in a random direction
    v = _rand((rows, width), "fp32", 21)
    loss = [float(((w.double() + s * v.double())[ids] * 3.0 * up.double()
                   * (ids != ids[0, 0])[..., None]).sum()) for s in (0.125, -0.125)]
    got = float((w.grad.double() * v.double()).sum())
    assert abs((loss[0] - loss[1]) / 0.25 - got) <= 1e-5 * float((w.grad * v).abs().sum())
    assert not ms.ops.embedding(ids, w.detach()).requires_grad


@pytest.mark.parametrize("rows,width,n", [(300, 72, 200), (5000, 136, 3000)])
def test_in_a_graph(rows, width, n):
    ids, g = _ids(n, rows, 22), _rand((n, width), "bf16", 23)
    w = _rand((rows, width), "bf16", 24)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(2):
            ms.ops.embedding(ids, w), ms.ops.embedding_grad(g, ids, rows)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, dw = ms.ops.embedding(ids, w), ms.ops.embedding_grad(g, ids, rows)
    for seed in range(30, 34):
        ids.copy_(_ids(n, rows, seed))
        g.copy_(_rand((n, width), "bf16", seed))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ms.ops.embedding(ids, w))
        assert torch.equal(dw, ms.ops.embedding_grad(g, ids, rows))


def test_refusals():
    w, ids = _rand((10, 8), "fp32", 25), torch.zeros(4, dtype=torch.int64, device=DEV)
    g = _rand((4, 8), "fp32", 26)
    with pytest.raises(TypeError, match="ids"):
        ms.ops.embedding(ids.float(), w)
    with pytest.raises(TypeError, match="weight"):
        ms.ops.embedding(ids, w.double())
    with pytest.raises(ValueError, match="weight"):
        ms.ops.embedding(ids, w[0])
    with pytest.raises(ValueError, match="no rows"):
        ms.ops.embedding(ids, w[:0])
    with pytest.raises(RuntimeError, match="cpu"):
        ms.ops.embedding(ids.cpu(), w)
    with pytest.raises(RuntimeError, match="cpu"):
        ms.ops.embedding(ids, w.cpu())
    with pytest.raises(ValueError, match="padding_idx"):
        ms.ops.embedding(ids, w, padding_idx=10)
    with pytest.raises(ValueError, match="grad"):
        ms.ops.embedding_grad(g[:3], ids, 10)
    with pytest.raises(ValueError, match="grad"):
        ms.ops.embedding_grad(g.view(-1), ids, 10)
    with pytest.raises(ValueError, match="rows"):
        ms.ops.embedding_grad(g, ids, -1)
    with pytest.raises(TypeError, match="grad"):
        ms.ops.embedding_grad(g.double(), ids, 10)
    with pytest.raises(RuntimeError, match="cpu"):
        ms.ops.embedding_grad(g.cpu(), ids, 10)


def test_an_error_that_earlier_work_left_is_not_taken_for_the_launchs():
    """The thread's last HIP error (here of a device number that there is not) is neither
    reported by the operators nor taken away."""
    rows, width, n = 3000, 64, 2000                      # three launches
    w, ids, g = _rand((rows, width), "fp32", 33), _ids(n, rows, 34), _rand((n, width), "fp32", 35)
    out, dw = torch.empty(n, width, device=DEV), torch.empty(rows, width, device=DEV)
    lib, hip = ctypes.CDLL(build.OPS_OUTPUT), ctypes.CDLL("libamdhip64.so.7")
    lib.ms_embedding_grad_workspace.restype = ctypes.c_int64
    i64, ptr, ref_of = ctypes.c_int64, ctypes.c_void_p, ctypes.byref
    size = lib.ms_embedding_grad_workspace(i64(n), i64(rows), i64(width))
    work = torch.empty(size, dtype=torch.uint8, device=DEV)
    table, grad = Rows(w.data_ptr(), rows, width, rows, 0, width, 0, 0), Rows(g.data_ptr(), n, width, n,
                                                                              0, width, 0, 0)
    tokens = Tokens(ids.data_ptr(), n, n, 0, 1, 1, 0)
    stream = ptr(torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    hip.hipGetLastError()
    bad = hip.hipSetDevice(9999)
    codes = [lib.ms_embedding(ref_of(tokens), ref_of(table), ctypes.c_float(1), ptr(out.data_ptr()),
                              stream),
             lib.ms_embedding_grad(ref_of(tokens), ref_of(grad), i64(rows), ctypes.c_float(1),
                                   i64(-1), ptr(dw.data_ptr()), ptr(work.data_ptr()), i64(size),
                                   stream)]
    left = hip.hipGetLastError()
    assert bad != 0 and codes == [0, 0] and left == bad
    assert torch.equal(out, w[ids]) and torch.equal(dw, ms.ops.embedding_grad(g, ids, rows))
