"""fp16 gradients of the loss without logits whose rows have gradients of very different size.

Tolerances.  Those of tests/test_gpu_ops_linear.py for rows of like gradients.  Beside them, dweight's
copy of hidden: a row is multiplied by a power of two s, such that for the row of the largest product of
gradient and hidden value the latter comes to 2^15 or more.  What underflows in the copy is off by
2^-25, which in hidden's own units is 2^-25 / s with 1 / s <= 2 B H 2^-15 / b, for a row of gradient b and
the largest gradient B and value H of any row: with the row's d that makes 2^-39 B H |d| / b.
"""

from __future__ import annotations

import pytest
import torch

import minispeed_amd as ms
from tests import ops_reference as ref
from tests.test_gpu_ops_linear import DEV, backward, check, make

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


@pytest.mark.parametrize("big,small", [(2.0 ** 12, 2.0 ** -12), (2.0 ** 8, 2.0 ** -10), (2.0 ** 12, 2.0 ** -4),
                                       (2.0 ** -2, 2.0 ** -12)])
@pytest.mark.parametrize("n,d", [(400, 32), (401, 37), (300, 1030)])
def test_words_that_only_rows_of_small_gradients_hold(big, small, n, d):
    """The last 60 words have logits of -60 in the rows of large gradients, so that nothing but the
    other rows makes their dweight."""
    h, w, t, gr, _ = make(n, d, 300, "fp16", n + d, ignored=0.0)
    few = torch.arange(n, device=DEV) % 2 == 1
    h[:, 0] = torch.where(few, -1.0, 1.0)
    w[:, 0] = 0.0
    w[240:, 0] = -60.0
    t = torch.where(few, 240 + t % 60, t % 240)
    gr = torch.where(few, small, big) * torch.sign(gr)
    r = ms.ops.linear_logprobs(h, w, t)
    dh, dw = ms.ops.linear_logprobs_grad(h, w, t, r.lse, gr)
    eh, ew, th, _ = backward(h, w, t, gr, None)
    ref.close(dh, eh, th)
    tol = torch.zeros_like(ew)
    for rows in (few, ~few):
        tol += backward(h[rows], w, t[rows], gr[rows], None)[3]
    p = torch.softmax(h.double() @ w.double().T, 1)
    p.scatter_add_(1, t[:, None], torch.ones(n, 1, device=DEV, dtype=torch.float64))
    copy = 2.0 ** -39 * big * h.abs().max().double() * p.sum(0)
    ref.close(dw, ew, tol + copy[:, None])
    # (of the oracle alone: zeros in the place of the small rows' part would be outside the tolerance)
    held = ew[240:].abs() > tol[240:] + copy[240:, None]
    assert bool(held.any(1)[t[few] - 240].all())


@pytest.mark.parametrize("size", [2.0 ** -20, 1.0, 2.0 ** 14])
def test_hidden_states_of_any_size(size):
    """The copy is lifted to fp16's largest numbers and does not pass them."""
    h, w, t, gr, gl = make(200, 72, 300, "fp16", 5)
    h[3, 5], h[7], h[9, 1] = 4.0, 0.0, -(4 - 2.0 ** -9)
    t[9] = 6
    # (4 x 2^14 would be infinity)
    h = (h.clamp(-4, 4).float() * size).clamp(-65504, 65504).half()
    w = (w / size).clamp(-6e4, 6e4).half() if size > 1 else w
    check(h, w, t, gr, gl)
    # (dweight within fp16's range)
    check(h, w, t, gr * 2.0 ** 12 / max(size, 1.0), gl)
