"""fp16 gradients of the loss without logits whose rows have gradients of very different size.

Tolerances: those of tests/test_gpu_ops_linear.py for a row by itself.
"""

from __future__ import annotations

import pytest
import torch

import minispeed_amd as ms
from tests import ops_reference as ref
from tests.test_gpu_ops_linear import DEV, backward, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [40, 2048, 20000])
@pytest.mark.parametrize("tiny", [1e-40, 1e-38, 2.0 ** -149, 1e-30])
def test_rows_of_next_to_no_gradient(n, tiny):
    """dweight among rows of 1 / n with some of subnormal numbers, which add nothing to it that
    could be seen: the tolerance is that of the ordinary rows alone."""
    h, w, t, _, _ = make(n, 64, 300, "fp16", n, ignored=0.0)
    gr = torch.full((n,), -1.0 / n, device=DEV)
    few = torch.arange(n, device=DEV) % 17 == 3
    gr[few] = -tiny
    r = ms.ops.linear_logprobs(h, w, t)
    dh, dw = ms.ops.linear_logprobs_grad(h, w, t, r.lse, gr)
    eh, ew, _, _ = backward(h, w, t, gr, None)
    _, _, th, tw = backward(h, w, t, gr.masked_fill(few, 0.0), None)
    ref.close(dw, ew, tw + few.sum() * tiny * h.abs().max())
    ref.close(dh, eh, th + tiny)


def test_rows_of_nothing_else():
    """Subnormal gradients alone, brought back by the scale of the logits' gradients' sums."""
    h, w, t, _, _ = make(50, 32, 70, "fp16", 3, ignored=0.0)
    gr = torch.full((50,), -1e-40, device=DEV)
    r = ms.ops.linear_logprobs(h, w, t)
    dh, dw = ms.ops.linear_logprobs_grad(h, w, t, r.lse, gr)
    assert not dh.any() and not dw.any()
