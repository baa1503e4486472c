"""The workspace of the loss without logits, counted on the CPU: what the library asks for is
enough for every choice of gradients, and stays near what the operator has to hold."""

from __future__ import annotations

import ctypes
import random

import pytest

from minispeed_amd import build
from tests.test_ops_abi import Rows, Tokens

P, I32, I64, F = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float
REF = ctypes.byref
BOTH, HIDDEN, WEIGHT = (1, 1), (1, 0), (0, 1)


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(build.OPS_OUTPUT)
    for name in ("ms_linear_logprobs_grad_workspace", "ms_linear_logprobs_grad_workspace_for"):
        getattr(lib, name).restype = I64
    return lib


def _rows(n, width, dtype, data=16):
    return Rows(data, n, width, max(n, 1), 0, width, dtype, 0)


def _query(lib, h, w):
    return lib.ms_linear_logprobs_grad_workspace(REF(h), REF(w))


def _takes(lib, h, w, wanted):
    return lib.ms_linear_logprobs_grad_workspace_for(REF(h), REF(w), *map(I32, wanted))


def _call(lib, h, w, wanted, size, ids=None):
    """Refusals only: with enough space it would launch."""
    n = h.n
    ids = ids or Tokens(16, n, max(n, 1), 0, 1, 1, 0)
    return lib.ms_linear_logprobs_grad(REF(h), REF(w), REF(ids), F(1), I64(-100), P(16), P(16), None,
                                       P(16 if wanted[0] else None), P(16 if wanted[1] else None), P(16),
                                       I64(size), None)


# (a lone gradient's own plan has more parts of k than the plan of both at each of these)
CUT = [(2048, 4096, 128256, 2), (16384, 768, 50257, 2), (4096, 5120, 32000, 2), (2048, 2048, 50257, 1),
       (1024, 2048, 50257, 0), (1196, 2224, 8141, 2), (121, 2176, 24197, 2), (1090, 576, 8059, 2),
       (512, 4096, 128256, 2), (2048, 768, 50257, 2)]


@pytest.mark.parametrize("n,d,v,dtype", CUT)
def test_one_gradient_alone_where_it_takes_more_than_both(lib, n, d, v, dtype):
    h, w = _rows(n, d, dtype), _rows(v, d, dtype)
    both, *alone = (_takes(lib, h, w, x) for x in (BOTH, HIDDEN, WEIGHT))
    assert max(alone) > both > 0
    assert _query(lib, h, w) == max(alone)
    for wanted, need in zip((BOTH, HIDDEN, WEIGHT), (both, *alone)):
        assert _call(lib, h, w, wanted, need - 1) == -2


def test_the_query_is_enough_for_every_choice_of_gradients(lib):
    rng = random.Random(11)
    log = lambda lo, hi: int(round(lo * (hi / lo) ** rng.random()))  # noqa: E731
    for _ in range(4000):
        n, d, v = log(1, 65536), log(1, 8192), log(1, 262144)
        if rng.random() < 0.5:
            n, d, v = n, -(-d // 64) * 64, v
        dtype = rng.randrange(3)
        h, w = _rows(n, d, dtype, rng.choice((16, 18 if dtype else 20))), _rows(v, d, dtype)
        query = _query(lib, h, w)
        for wanted in (BOTH, HIDDEN, WEIGHT):
            need = _takes(lib, h, w, wanted)
            assert 0 < need <= query
            if rng.random() < 0.1:
                assert _call(lib, h, w, wanted, need - 1) == -2


def test_refused_sizes(lib):
    w = _rows(10, 16, 1)
    assert _takes(lib, _rows(4, 17, 1), w, BOTH) == -1 and _takes(lib, _rows(4, 16, 2), w, HIDDEN) == -1
    assert lib.ms_linear_logprobs_grad_workspace_for(None, REF(w), I32(1), I32(1)) == -1
    assert _query(lib, _rows(4, 17, 1), w) == -1
    assert _takes(lib, _rows(0, 16, 1), w, BOTH) == 0 and _takes(lib, _rows(4, 16, 1), w, (0, 0)) == 0


def _up(x, to):
    return -(-x // to) * to


def _terms(n, d, v, dtype):
    """What the operator holds whatever the parts of its sums: (bytes, columns of a piece, pieces, bytes of a
    copy of hidden).  Operands on 16 bytes."""
    size, planes = (2, 1) if dtype else (4, 1)
    if dtype == 0 and n > 384 and n * d * v > 1 << 29:
        size, planes = 2, 3
    most = min(max((512 << 20) // (n * size * planes) // 256 * 256, 256), 1 << 20)
    pieces = -(-v // most)
    piece = _up(-(-v // pieces), 256)
    held = _up(16 * n, 256) + 256 + _up(_up(n * piece, 128) * planes * size, 256)
    if planes == 3:
        held += sum(_up(_up(rows * d, 128) * 6, 256) for rows in (n, v))
    return held, min(piece, v), pieces, _up(n * d * 2, 256) + 2048 if dtype == 1 else 0


PARTS = (1, 2, 3, 4, 6, 8, 16, 32, 64)


def test_the_workspace_by_its_terms(lib):
    """Row numbers, a piece of d, the copies, and whole sets of sums in 32 bits, within what the
    documentation states."""
    rng = random.Random(12)
    log = lambda lo, hi: int(round(lo * (hi / lo) ** rng.random()))  # noqa: E731
    cases = [(8192, 2048, 50257, 1), (16384, 768, 50257, 2), (2 ** 20, 64, 128256, 2), (4, 4096, 128256, 2)]
    cases += [(log(1, 200000), _up(log(8, 16384), 8), log(64, 300000), rng.randrange(3)) for _ in range(3000)]
    for n, d, v, dtype in cases:
        h, w = _rows(n, d, dtype), _rows(v, d, dtype)
        held, columns, pieces, copy = _terms(n, d, v, dtype)
        of_h = {0} if pieces == 1 else set()
        of_h |= {_up(s * n * d * 4, 256) for s in PARTS if s > 1 or pieces > 1}
        of_w = {0} | {_up(s * columns * d * 4, 256) for s in PARTS if s > 1}
        one = n * d * 4 if pieces > 1 else 0
        for wanted in (BOTH, HIDDEN, WEIGHT):
            sums = _takes(lib, h, w, wanted) - held - (copy if wanted[1] else 0)
            if wanted == HIDDEN:
                assert sums in of_h
            elif wanted == WEIGHT:
                assert sums in of_w
            else:
                assert any(sums - x in of_w for x in of_h)
            more = sums - (one if wanted[0] else 0)
            assert more <= (128 << 20 if dtype and wanted == BOTH else 1280 << 20)
