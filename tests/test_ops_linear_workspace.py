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
