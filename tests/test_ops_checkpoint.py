"""checkpoint8 on the host: its autograd, with tensors that no kernel touches (what is
not on a GPU is kept as it is)."""

from __future__ import annotations

import pytest
import torch

import minispeed_amd as ms


def test_parameters_get_gradients_when_no_argument_requires_one():
    layer = torch.nn.Linear(4, 3)
    x = torch.arange(8.0).view(2, 4)
    y = ms.ops.checkpoint8(layer, x)
    assert y.requires_grad
    y.sum().backward()
    assert torch.equal(layer.weight.grad, x.sum(0).expand(3, 4))
    assert not ms.ops.checkpoint8(lambda a: a * 2, x).requires_grad


@pytest.mark.parametrize("wrap", [lambda y: [y], lambda y: {"y": y}, lambda y: (y, (y, y)),
                                  lambda y: (y, [y])])
def test_results_whose_gradients_would_be_lost_are_refused(wrap):
    x = torch.ones(3, requires_grad=True)
    with pytest.raises(TypeError, match="tuple"):
        ms.ops.checkpoint8(lambda a: wrap(a * 2), x)
    y, n, none, sizes = ms.ops.checkpoint8(lambda a: (a * 2, 7, None, [1, 2]), x)
    assert n == 7 and none is None and sizes == [1, 2]
    y.sum().backward()
    assert torch.equal(x.grad, torch.full((3,), 2.0))
