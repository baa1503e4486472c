"""Layer norms of rows that hold one number, up to the type's lowest value, as padding does: their
deviation from the mean is zero, so all results are those of rows of zeros, bit for bit.  (The numbers
have 8 bits, so that sums over a row are exact in 32.)"""

from __future__ import annotations

import pytest
import torch

import minispeed_amd as ms
from tests.ops_reference import DTYPES

pytestmark = pytest.mark.gpu
DEV = "cuda"
LOWEST = float(torch.finfo(torch.bfloat16).min)
CASES = [(dtype, value) for dtype in ("bf16", "fp32") for value in (LOWEST, -LOWEST, -1.25 * 2.0 ** 122, 2.0 ** 120, 3.0)]
CASES += [("fp16", -65280.0), ("fp16", 3.0)]


def _operands(width, dtype, gates):
    g = torch.Generator(device=DEV).manual_seed(width)
    def randn(*size):
        return torch.randn(*size, generator=g, device=DEV).to(DTYPES[dtype])
    return [randn(3, 7, width) for _ in range(4)], [randn(width) for _ in range(4)], \
        randn(3, 1, width) if gates else None


@pytest.mark.parametrize("width", [1, 7, 8, 96, 768, 1000, 2048, 2049, 5000, 10000, 16384])
@pytest.mark.parametrize("dtype,value", CASES)
def test_norm(dtype, value, width):
    (x, dy, _, _), (w, b, _, _), _ = _operands(width, dtype, False)
    results = []
    for fill in (value, 0.0):
        x = x.clone()
        x[0, 3:], x[2, 6] = fill, fill
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        y = ms.ops.norm(*leaves, kind="layer")
        y.backward(dy)
        results.append([y, *(t.grad for t in leaves)])
    for got, want in zip(*results):
        assert torch.isfinite(got).all() and torch.equal(got, want)


@pytest.mark.parametrize("gates", [False, True])
@pytest.mark.parametrize("width", [1, 7, 768, 1000, 2048, 5000, 10000])
@pytest.mark.parametrize("dtype,value", CASES)
def test_residual_norm(dtype, value, width, gates):
    (x, block, dr, dy), weights, gate = _operands(width, dtype, gates)
    results = []
    for fill in (value, 0.0):
        block = block.clone()
        block[0, 3:], block[2, 6] = fill, fill
        leaves = [t.clone().requires_grad_() for t in (x, block, *weights, *([gate] if gates else []))]
        r = ms.ops.residual_norm(*leaves, scale=0.75, kind="layer")
        torch.autograd.backward([r.residual, r.out], [dr, dy])
        results.append([r.residual, r.out, *(t.grad for t in leaves)])
    for got, want in zip(*results):
        assert torch.isfinite(got).all() and torch.equal(got, want)
