"""Operands of more than one type, as ``torch.autocast`` gives them."""

from __future__ import annotations

import torch

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def of_one_type(tensors, dtype=None):
    """The tensors (``None`` among them), where their types differ cast to ``dtype``, by default
    autocast's own.  For calls under autocast: elsewhere what differs is refused."""
    types = {t.dtype for t in tensors if t is not None}
    if len(types) == 1 or not types.issubset(_FLOATS):
        return tensors
    dtype = dtype or torch.get_autocast_dtype("cuda")
    return tuple(t if t is None else t.to(dtype) for t in tensors)
