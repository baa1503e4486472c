"""The cast of operands of several types, on the CPU."""

from __future__ import annotations

import torch

from minispeed_amd.ops._types import of_one_type


def test_only_what_differs_is_cast(monkeypatch):
    a, b = torch.zeros(2), torch.zeros(3, dtype=torch.float16)
    monkeypatch.setattr(torch, "get_autocast_dtype", lambda device: torch.bfloat16)
    out = of_one_type((a, None, b))
    assert out[1] is None and out[0].dtype == out[2].dtype == torch.bfloat16
    assert all(t.dtype == torch.float32 for t in of_one_type((a, b), torch.float32))
    assert of_one_type((a, a))[0] is a and of_one_type((b, None), torch.float32)[0] is b
    # (what the kernels do not take is left for them to refuse)
    for dtype in (torch.int64, torch.float64):
        other = torch.zeros(2, dtype=dtype)
        assert of_one_type((a, other))[1] is other
