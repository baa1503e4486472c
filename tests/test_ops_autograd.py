"""What the operators say to derivatives that they do not have, before anything is launched."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import minispeed_amd as ms

ops = ms.ops


def _calls(x):
    ids = torch.zeros(4, dtype=torch.int64)
    row = torch.zeros(4)
    held = ops.Checkpoint8(torch.zeros(32, dtype=torch.int8), torch.ones(1, dtype=torch.uint8),
                           (4, 8), torch.float32)
    plain = x.detach()
    yield lambda: ops.embedding(ids, x)
    yield lambda: ops.embedding_grad(x, ids, 10)
    yield lambda: ops.token_logprobs(x, ids)
    yield lambda: ops.token_logprobs_grad(x, ids, row, row)
    yield lambda: ops.token_logprobs_grad(plain, ids, x[:, 0], row)
    yield lambda: ops.token_logprobs_grad(plain, ids, row, x[:, 0])
    yield lambda: ops.token_logprobs_grad(plain, ids, row, row, x[:, 0], x[:, 0])
    yield lambda: ops.pack8(x)
    yield lambda: ops.activation8(x)
    yield lambda: ops.activation8(plain, "swiglu", up=x)
    yield lambda: ops.activation8_grad((held,), x)


@pytest.mark.parametrize("k", range(11))
def test_forward_mode_is_refused_and_not_dropped(k):
    with forward_ad.dual_level():
        x = forward_ad.make_dual(torch.zeros(4, 8), torch.ones(4, 8))
        with pytest.raises(NotImplementedError, match="forward"):
            list(_calls(x))[k]()
        with forward_ad._set_fwd_grad_enabled(False), pytest.raises(RuntimeError, match="cpu"):
            list(_calls(x))[k]()
