"""One gradient of the loss without logits by itself (a frozen head, or frozen hidden states), at
sizes where its own plan takes more space than that of both, against 64-bit sums with the
tolerances of tests/test_gpu_ops_linear.py."""

from __future__ import annotations

import ctypes

import pytest
import torch

import minispeed_amd as ms
from minispeed_amd import build
from tests import ops_reference as ref
from tests.test_gpu_ops_linear import DEV, backward, make
from tests.test_ops_abi import Rows, Tokens

pytestmark = pytest.mark.gpu
TYPES = {"fp32": 0, "fp16": 1, "bf16": 2}
# (n, width, vocab, type): more for dhidden alone, or for dweight alone, or each, than for both
SIZES = [(121, 2176, 24197, "bf16"), (1090, 576, 8059, "bf16"), (1196, 2224, 8141, "bf16"),
         (2986, 131, 3493, "bf16"), (6539, 65, 3233, "fp16"), (474, 131, 21273, "fp16"),
         (587, 64, 14418, "fp32"), (1154, 144, 3245, "fp32")]


@pytest.mark.parametrize("n,d,v,dtype", SIZES)
def test_within_its_workspace(n, d, v, dtype):
    """The C entry with exactly the bytes that the call takes, and guard bytes behind them."""
    lib = ctypes.CDLL(build.OPS_OUTPUT)
    P, I32, I64, F, by = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float, ctypes.byref
    lib.ms_linear_logprobs_grad_workspace_for.restype = I64
    lib.ms_linear_logprobs_grad_workspace.restype = I64
    h, w, t, gr, gl = make(n, d, v, dtype, n)
    hr, wr = (Rows(x.data_ptr(), len(x), d, len(x), 0, d, TYPES[dtype], 0) for x in (h, w))
    ids = Tokens(t.data_ptr(), n, n, 0, 1, 1, 0)
    lse = ms.ops.linear_logprobs(h, w, t).lse
    eh, ew, th, tw = backward(h, w, t, gr, gl)
    guard = 1 << 20
    for wanted in ((1, 0), (0, 1), (1, 1)):
        need = lib.ms_linear_logprobs_grad_workspace_for(by(hr), by(wr), *map(I32, wanted))
        assert 0 < need <= lib.ms_linear_logprobs_grad_workspace(by(hr), by(wr))
        work = torch.full((need + guard,), 77, dtype=torch.uint8, device=DEV)
        dh, dw = torch.full_like(h, 3.0), torch.full_like(w, 3.0)
        assert lib.ms_linear_logprobs_grad(
            by(hr), by(wr), by(ids), F(1), I64(-100), P(lse.data_ptr()), P(gr.data_ptr()),
            P(gl.data_ptr()), P(dh.data_ptr() if wanted[0] else None),
            P(dw.data_ptr() if wanted[1] else None), P(work.data_ptr()), I64(need),
            P(torch.cuda.current_stream().cuda_stream)) == 0
        assert bool((work[need:] == 77).all())
        if wanted[0]:
            ref.close(dh, eh, th, "dhidden")
        else:
            assert bool((dh == 3.0).all())
        if wanted[1]:
            ref.close(dw, ew, tw, "dweight")
        else:
            assert bool((dw == 3.0).all())


@pytest.mark.parametrize("n,d,v,dtype", SIZES)
@pytest.mark.parametrize("need", [(True, False), (False, True)])
def test_frozen_operands(n, d, v, dtype, need):
    h, w, t, gr, gl = make(n, d, v, dtype, n + 1)
    a, b = h.clone().requires_grad_(need[0]), w.clone().requires_grad_(need[1])
    r = ms.ops.linear_logprobs(a, b, t)
    ((r.logprob * gr).sum() + (r.lse * gl).sum()).backward()
    assert (a.grad is None) != need[0] and (b.grad is None) != need[1]
    eh, ew, th, tw = backward(h, w, t, gr, gl)
    if need[0]:
        ref.close(a.grad, eh, th, "dhidden")
    else:
        ref.close(b.grad, ew, tw, "dweight")


@pytest.mark.parametrize("n,d,v,dtype", [(1090, 576, 8059, "bf16"), (2986, 131, 3493, "fp16"),
                                         (587, 64, 14418, "fp32")])
@pytest.mark.parametrize("wanted", [(True, False), (False, True)])
def test_in_a_graph_and_beside_another_stream(n, d, v, dtype, wanted):
    h, w, t, gr, gl = make(n, d, v, dtype, n)
    native = ms.ops._native

    def step():
        r = ms.ops.linear_logprobs(h, w, t)
        return [x for x in native.linear_logprobs_grad(h, w, t, r.lse, gr, gl, 1.0, -100, *wanted)
                if x is not None]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(3):
        new = make(n, d, v, dtype, 100 + seed)
        h.copy_(new[0])
        gr.copy_(new[3] * 10.0 ** -seed)
        side.wait_stream(torch.cuda.current_stream())
        graph.replay()
        with torch.cuda.stream(side):
            beside = step()
        want = step()
        torch.cuda.synchronize()
        assert len(out) == 1 and torch.isfinite(want[0]).all()
        assert torch.equal(out[0], want[0]) and torch.equal(beside[0], want[0])
