"""The block and head operators on the CPU: what their C entries and their Python entry points
refuse, before anything is launched."""

from __future__ import annotations

import ctypes

import pytest
import torch
from torch.autograd import forward_ad

import minispeed_amd as ms
from minispeed_amd import build
from tests.test_ops_abi import Rows, Tokens

P, I32, I64, F = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float
REF = ctypes.byref


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(build.OPS_OUTPUT)
    for name in ("ms_linear_logprobs_workspace", "ms_linear_logprobs_grad_workspace",
                 "ms_norm_grad_workspace", "ms_position_bias_grad_workspace"):
        getattr(lib, name).restype = I64
    return lib


def _rows(n, width, dtype=1, data=16):
    return Rows(data, n, width, max(n, 1), 0, width, dtype, 0)


def test_linear_logprobs(lib):
    h, w, ids = _rows(4, 16), _rows(10, 16), Tokens(16, 4, 4, 0, 1, 1, 0)
    need = lib.ms_linear_logprobs_workspace(REF(h), REF(w))
    more = lib.ms_linear_logprobs_grad_workspace(REF(h), REF(w))
    assert need > 0 and more > 0

    def call(h=h, w=w, ids=ids, lp=16, lse=16, ws=16, size=need):
        return lib.ms_linear_logprobs(REF(h), REF(w), REF(ids), F(1), I64(-100), P(lp), P(lse), P(ws),
                                      I64(size), None)

    def back(h=h, w=w, ids=ids, lse=16, dh=16, dw=16, ws=16, size=more):
        return lib.ms_linear_logprobs_grad(REF(h), REF(w), REF(ids), F(1), I64(-100), P(lse), P(16), None,
                                           P(dh), P(dw), P(ws), I64(size), None)

    for f in (call, back):
        assert f(h=_rows(4, 17)) == -1 and f(h=_rows(4, 16, 2)) == -1 and f(w=_rows(0, 16)) == -1
        assert f(h=_rows(4, 0), w=_rows(10, 0)) == -1 and f(h=_rows(5, 16)) == -1
        assert f(h=_rows(4, 2 ** 20 + 8), w=_rows(10, 2 ** 20 + 8)) == -1
        assert f(h=_rows(4, 16, 5), w=_rows(10, 16, 5)) == -1 and f(h=_rows(4, 16, data=None)) == -1
        assert f(lse=None) == -1 and f(ws=24) == -2 and f(ws=None) == -2
        assert f(size=(need if f is call else more) - 1) == -2
        most = _rows(2 ** 31 - 1, 2 ** 20)
        assert f(h=most, w=_rows(2 ** 31 - 1, 2 ** 20), ids=Tokens(16, 2 ** 31 - 1, 2 ** 31 - 1, 0, 1, 1, 0)) < 0
    assert call(lp=None) == -1
    assert back(dh=None, dw=None) == 0
    empty = Tokens(None, 0, 1, 0, 0, 1, 0)
    assert call(h=_rows(0, 16), ids=empty) == 0
    assert back(h=_rows(0, 16), ids=empty, dw=None) == 0
    assert lib.ms_linear_logprobs_workspace(REF(_rows(4, 17)), REF(w)) == -1
    assert lib.ms_linear_logprobs_workspace(None, REF(w)) == -1


def test_a_piece_of_the_vocabulary_bounds_the_workspace(lib):
    """Backward: no more than 512 MiB or 256 words of d, whatever the sizes, beside sums of
    dhidden."""
    for n, d, v, dtype in ((8192, 2048, 50257, 1), (16384, 768, 50257, 2), (2 ** 20, 64, 128256, 2),
                           (4, 4096, 128256, 2)):
        need = lib.ms_linear_logprobs_grad_workspace(REF(_rows(n, d, dtype)), REF(_rows(v, d, dtype)))
        piece = max(512 << 20, n * 256 * 2)
        assert need <= piece + 600 * 4096 * 4 * max(1, n * d // 65536) + n * (d * 2 + 16) + 4096


def test_norm(lib):
    x, y, thin = _rows(6, 16), _rows(6, 16), _rows(6, 15)

    def call(x=x, block=y, kind=1, w=16, b=16, bw=16, bb=16, gate=16, gates=2, nxt=16, out=16):
        return lib.ms_norm(REF(x), REF(block) if block else None, I32(kind), P(w), P(b), P(bw), P(bb),
                           P(gate), I64(gates), F(1), F(1e-5), P(nxt), P(out), None, None)

    assert call(block=thin) == -1 and call(kind=2) == -1 and call(w=None) == -1
    assert call(kind=0) == -1 and call(bw=None) == -1 and call(block=None) == -1
    assert call(gates=4) == -1 and call(gates=0) == -1 and call(gate=None) == -1
    assert call(nxt=None) == -1 and call(out=None) == -1
    assert call(x=_rows(6, 16385), block=_rows(6, 16385)) == -1
    assert call(x=_rows(0, 16, data=None), block=_rows(0, 16, data=None)) == 0
    size = lambda *a: lib.ms_norm_grad_workspace(I64(a[0]), I64(a[1]), I32(1), I32(1), I32(1), I64(a[2]))  # noqa: E731
    assert size(6, 16, 2) > 0 and size(6, 16, 4) == -1 and size(-1, 16, 0) == -1 and size(6, 16385, 0) == -1
    need = size(6, 16, 2)

    def back(dout=x, dnext=y, nxt=x, stats=16, block=y, kind=1, bw=16, bb=16, gate=16, gates=2, dx=16,
             db=16, dw=16, dbias=16, dbw=16, dbb=16, dg=16, ws=16, ws_size=need):
        opt = lambda r: REF(r) if r else None  # noqa: E731
        return lib.ms_norm_grad(opt(dout), opt(dnext), REF(nxt), P(stats), opt(block), I32(kind), P(16),
                                P(bw), P(bb), P(gate), I64(gates), F(1), P(dx), P(db), P(dw), P(dbias),
                                P(dbw), P(dbb), P(dg), P(ws), I64(ws_size), None)

    assert back(dout=None, dnext=None) == -1 and back(dout=thin) == -1 and back(dnext=thin) == -1
    assert back(stats=None) == -1 and back(dx=None) == -1 and back(db=None) == -1 and back(dw=None) == -1
    assert back(dbw=None) == -1 and back(dg=None) == -1 and back(kind=0) == -1
    assert back(bw=None, bb=None) == -1 and back(gate=None, gates=0) == -1 and back(gates=5) == -1
    assert back(ws=8) == -2 and back(ws=None) == -2 and back(ws_size=need - 1) == -2


def test_position_bias(lib):
    def call(table=16, dtype=1, buckets=32, heads=4, q=5, k=6, first=0, far=128, causal=0, out=16):
        return lib.ms_position_bias(P(table), I32(dtype), I64(buckets), I64(4), I64(1), I64(heads), I64(q),
                                    I64(k), I64(first), I64(far), I32(causal), P(out), None)

    def back(grad=16, dtype=1, batch=2, heads=4, q=5, k=6, first=0, buckets=32, far=128, causal=0, out=16,
             ws=16, size=1 << 40):
        return lib.ms_position_bias_grad(P(grad), I32(dtype), I64(batch), I64(120), I64(heads), I64(30), I64(q),
                                         I64(6), I64(k), I64(first), I64(buckets), I64(far), I32(causal),
                                         P(out), P(ws), I64(size), None)

    for f in (call, back):
        assert f(dtype=3) == -1 and f(buckets=2) == -1 and f(buckets=33) == -1 and f(buckets=514) == -1
        assert f(far=8) == -1 and f(far=2 ** 31) == -1 and f(heads=-1) == -1 and f(q=-1) == -1
        assert f(k=2 ** 31) == -1 and f(first=2 ** 41) == -1 and f(out=None) == -1
        assert f(heads=2 ** 31 - 1, q=2 ** 31 - 1, k=2 ** 31 - 1) == -1
        assert f(heads=0) == 0
    assert call(table=None) == -1 and call(q=0) == 0 and call(k=0) == 0
    assert back(grad=None) == -1 and back(batch=-1) == -1 and back(ws=8) == -2 and back(ws=None) == -2
    size = lib.ms_position_bias_grad_workspace(I32(1), I64(32), I64(2), I64(4), I64(5), I64(6))
    assert size > 0 and back(size=size - 1) == -2
    # more blocks than one launch has
    assert call(heads=2 ** 20, q=2 ** 14, k=2 ** 12) == -1


def _calls(x):
    ids, row, plain = torch.zeros(4, dtype=torch.int64), torch.zeros(4), x.detach()
    w, stats = torch.zeros(8), torch.zeros(4, 2)
    yield lambda: ms.ops.linear_logprobs(x, plain, ids)
    yield lambda: ms.ops.linear_logprobs(plain, x, ids)
    yield lambda: ms.ops.linear_logprobs_grad(plain, plain, ids, x[:, 0], row)
    yield lambda: ms.ops.linear_logprobs_grad(plain, plain, ids, row, x[:, 0])
    yield lambda: ms.ops.linear_logprobs_grad(plain, plain, ids, row, row, x[:, 0])
    yield lambda: ms.ops.norm(x, w)
    yield lambda: ms.ops.residual_norm(x, plain, w)
    yield lambda: ms.ops.residual_norm_grad(plain, plain, x, stats, plain, w)
    yield lambda: ms.ops.position_bias(x, 3, 3)
    yield lambda: ms.ops.position_bias_grad(x[None], 8)


COUNT = 10


@pytest.mark.parametrize("k", range(COUNT))
def test_cpu_tensors_and_forward_mode_are_refused(k):
    assert len(list(_calls(torch.zeros(4, 8)))) == COUNT
    with pytest.raises(RuntimeError, match="cpu"):
        list(_calls(torch.zeros(4, 8)))[k]()
    with forward_ad.dual_level():
        x = forward_ad.make_dual(torch.zeros(4, 8), torch.ones(4, 8))
        with pytest.raises(NotImplementedError, match="forward"):
            list(_calls(x))[k]()


@pytest.mark.parametrize("kind", ["RMS", None, 0])
def test_an_unknown_norm_is_refused(kind):
    with pytest.raises(ValueError, match="norm"):
        ms.ops.norm(torch.zeros(4, 8), torch.zeros(8), kind=kind)
