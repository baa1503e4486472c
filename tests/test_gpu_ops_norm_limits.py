"""The norms' gradients at the largest number of rows, 2^31 - 1, of one value each.  All rows are
one row expanded, so every result is one number: with residual 1, deviation 2 and gradients of 1,
v = 1/2 and dresidual = 1 + (1 - v^2) / 2 = 1.375, exactly in every type."""

from __future__ import annotations

import pytest
import torch

import minispeed_amd as ms

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _all(x, value):
    """Whether all values are `value`, looked at 2^28 at a time."""
    flat = x.reshape(-1)
    return all(bool((flat[k:k + 2 ** 28] == value).all()) for k in range(0, flat.numel(), 2 ** 28))


@pytest.mark.parametrize("gates,each", [(0, 2 ** 31 - 1), (3, 715827882), (2147483, 1000), (2 ** 31 - 1, 1),
                                        (0, 2 ** 31 - 2049)])
def test_the_largest_number_of_rows(gates, each):
    one = torch.ones(1, 1, 1, dtype=torch.bfloat16, device=DEV)
    n = max(gates, 1) * each
    rows = one.expand(max(gates, 1), each, 1)
    stats = torch.tensor([0.0, 0.5], device=DEV).expand(max(gates, 1), each, 2)
    gate = one.expand(gates, 1, 1) if gates else None
    g = ms.ops.residual_norm_grad(rows, rows, rows, stats, rows, one[0, 0], gate=gate, scale=2.0)
    assert g.residual.shape == rows.shape and _all(g.residual, 1.375)
    assert _all(g.block, 2.75)
    # sums of n equal terms in fp32: partial sums of up to 2^20 terms, 4096 of them, each addition
    # off by 2^-24 of the sum
    tol = (2.0 ** 20 + 2.0 ** 12) * 2.0 ** -24 + 2.0 ** -8
    assert abs(float(g.weight) - 0.5 * n) <= tol * 0.5 * n
    if gates:
        assert g.gate.shape == (gates, 1, 1)
        assert bool(((g.gate.double() - 2.75 * each).abs() <= tol * 2.75 * each).all())
