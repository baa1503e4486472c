"""The block and head operators with the operands of several types that torch.autocast gives them:
the same bits as casts written out, gradients in the leaves' types; refused without autocast."""

from __future__ import annotations

import pytest
import torch

import minispeed_amd as ms

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _randn(*shape, seed, dtype=torch.float32):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, generator=g, device=DEV).to(dtype).requires_grad_()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("wide", ["weight", "hidden"])
def test_linear_logprobs(dtype, wide):
    types = (dtype, torch.float32) if wide == "weight" else (torch.float32, dtype)
    h, w = _randn(70, 40, seed=1, dtype=types[0]), _randn(300, 40, seed=2, dtype=types[1])
    t = torch.arange(70, device=DEV) * 4
    with pytest.raises(TypeError, match="dtype"):
        ms.ops.linear_logprobs(h, w, t)
    with torch.autocast("cuda", dtype=dtype):
        got = ms.ops.linear_logprobs(h, w, t)
    (-got.logprob.mean() + 0.01 * (got.lse ** 2).mean()).backward()
    grads, h.grad, w.grad = (h.grad, w.grad), None, None
    want = ms.ops.linear_logprobs(h.to(dtype), w.to(dtype), t)
    (-want.logprob.mean() + 0.01 * (want.lse ** 2).mean()).backward()
    assert all(torch.equal(a, b) for a, b in zip((*got, *grads), (*want, h.grad, w.grad)))
    assert (grads[0].dtype, grads[1].dtype) == types and torch.isfinite(w.grad).all()


def test_operands_of_one_type_are_not_cast():
    h, w, t = _randn(9, 16, seed=3), _randn(20, 16, seed=4), torch.arange(9, device=DEV)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got, y = ms.ops.linear_logprobs(h, w, t), ms.ops.norm(h.half(), w[0].half())
    assert torch.equal(got.lse, ms.ops.linear_logprobs(h, w, t).lse) and y.dtype == torch.float16


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_norms(dtype):
    x, out = _randn(3, 5, 48, seed=5), _randn(3, 5, 48, seed=6, dtype=dtype)
    w, b, bw, gate = (_randn(48, seed=k) for k in range(7, 11))
    with pytest.raises(TypeError, match="dtype"):
        ms.ops.residual_norm(x, out, w, b, bw, gate=gate, kind="layer")
    with pytest.raises(TypeError, match="dtype"):
        ms.ops.norm(out, w)
    leaves = (x, out, w, b, bw, gate)

    def run(cast):
        r = ms.ops.residual_norm(x, out.float() if cast else out, w, b, bw, gate=gate, kind="layer")
        y = ms.ops.norm(out.float() if cast else out, w)
        (r.residual.square().sum() + r.out.sum() + y.square().sum()).backward()
        grads = [p.grad for p in leaves]
        for p in leaves:
            p.grad = None
        return [*r, y, *grads]

    with torch.autocast("cuda", dtype=dtype):
        got = run(False)
    want = run(True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert got[0].dtype == got[1].dtype == torch.float32
    assert [g.dtype for g in got[-6:]] == [p.dtype for p in leaves]


def test_a_step_of_a_model_under_autocast():
    """Parameters in 32 bits, products in 16: the operators behind torch's own."""
    d, v = 64, 120
    table, head = _randn(v, d, seed=11), _randn(d, d, seed=12)
    w1, w2 = (torch.ones(d, device=DEV, requires_grad=True) for _ in range(2))
    ids = torch.arange(40, device=DEV).view(4, 10)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        x = ms.ops.embedding(ids, table)
        y = ms.ops.norm(x, w1)
        r = ms.ops.residual_norm(x, torch.nn.functional.linear(y, head), w2)
        loss = -ms.ops.linear_logprobs(torch.nn.functional.linear(r.out, head), table, ids).logprob.mean()
    loss.backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() and p.grad.any()
               for p in (table, head, w1, w2))
