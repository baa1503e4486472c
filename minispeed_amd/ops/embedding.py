"""Token embedding with scaling, and its gradient by sorted tokens."""

from __future__ import annotations

from typing import Optional

import torch

from . import _native


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, padding_idx):
        ctx.save_for_backward(ids)
        ctx.rows, ctx.scale, ctx.padding_idx = weight.shape[0], scale, padding_idx
        return _native.embedding(ids, weight, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        ids, = ctx.saved_tensors
        return None, _native.embedding_grad(grad, ids, ctx.rows, ctx.scale,
                                            ctx.padding_idx), None, None


def _padding(padding_idx: Optional[int], rows: int) -> int:
    if padding_idx is None:
        return -1
    if not -rows <= padding_idx < rows:
        raise ValueError(f"padding_idx is {padding_idx}, expected an index into {rows} rows")
    return padding_idx % rows


def embedding(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0,
              padding_idx: Optional[int] = None) -> torch.Tensor:
    """``scale * weight[ids]``, computed in 32 bits and rounded once.

    ``ids`` (int64 or int32, any shape and strides) selects rows of ``weight``
    (``[rows, width]``, float32 / float16 / bfloat16).  The gradient of
    ``weight`` is that of :func:`embedding_grad`; tokens equal to
    ``padding_idx`` add nothing to it.  An id outside ``[0, rows)`` gives a row
    of NaN and no gradient: checking the ids on the host would wait for the
    device.
    """
    skip = -1 if padding_idx is None else _padding(padding_idx, weight.shape[0])
    if weight.requires_grad and torch.is_grad_enabled():
        return _Embedding.apply(ids, weight, scale, skip)
    return _native.embedding(ids, weight, scale)


def embedding_grad(grad: torch.Tensor, ids: torch.Tensor, rows: int, scale: float = 1.0,
                   padding_idx: Optional[int] = None) -> torch.Tensor:
    """The gradient ``[rows, width]`` of an embedding table.

    ``grad`` (``[*ids.shape, width]``) is the gradient of the embedding's output.
    Row ``v`` is ``scale`` times the sum of the rows of ``grad`` whose id is
    ``v``, added in 32 bits in an order that follows from ``ids``, the sizes and
    the type, and rounded once: the same inputs give the same bits.  The whole table is
    written; rows without tokens are zeros.
    """
    return _native.embedding_grad(grad, ids, rows, scale, _padding(padding_idx, rows))
