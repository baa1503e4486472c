"""Learned relative position bias of attention, a table over buckets of distances."""

from __future__ import annotations

from typing import Optional

import torch

from . import _native


class _PositionBias(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, queries, keys, first, max_distance, causal):
        ctx.buckets, ctx.args = table.shape[0], (first, max_distance, causal)
        return _native.position_bias(table, queries, keys, first, max_distance, causal)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        return (_native.position_bias_grad(grad, ctx.buckets, *ctx.args),) + (None,) * 5


def position_bias(table: torch.Tensor, queries: int, keys: int, first: Optional[int] = None,
                  max_distance: int = 128, causal: bool = False) -> torch.Tensor:
    """``bias[h, i, j] = table[bucket(j - i - first), h]``, as ``[heads, queries, keys]``.

    ``table`` is ``[buckets, heads]`` (float32 / float16 / bfloat16, up to 512 buckets).  Query
    ``i`` stands at position ``first + i`` of the keys; by default the queries are the last
    ones, so that one new token after a cache has ``queries=1``.  The first half of a side's
    buckets tell distances one by one; the others widen in equal ratios up to
    ``max_distance``, and what is further shares the last.  Half of the buckets are for keys
    behind the query, after those for keys up to it; with ``causal=True`` all are
    for keys up to it, and the others get ``-inf``, so that the result is an attention mask.

    The gradient of ``table`` is that of :func:`position_bias_grad`.
    """
    first = keys - queries if first is None else first
    if table.requires_grad and torch.is_grad_enabled():
        return _PositionBias.apply(table, queries, keys, first, max_distance, causal)
    return _native.position_bias(table, queries, keys, first, max_distance, causal)


def position_bias_grad(grad: torch.Tensor, buckets: int, first: Optional[int] = None,
                       max_distance: int = 128, causal: bool = False) -> torch.Tensor:
    """The gradient ``[buckets, heads]`` of a table, given that of the bias.

    ``grad`` is ``[..., heads, queries, keys]``: sequences that shared the bias are summed
    here too.  Sums are made in 32 bits in an order that follows from the sizes and rounded
    once; with ``causal=True`` what lies at keys behind the query is not looked at.
    """
    if first is None:
        if grad.dim() < 3:
            raise ValueError(f"grad has shape {tuple(grad.shape)}, expected [..., heads, queries, keys]")
        first = grad.shape[-1] - grad.shape[-2]
    return _native.position_bias_grad(grad, buckets, first, max_distance, causal)
