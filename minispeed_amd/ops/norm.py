"""Norms before and after a block, with its gate, residual scale and residual sum."""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _native
from ._types import of_one_type

KINDS = {"rms": 0, "layer": 1}


class ResidualNorm(NamedTuple):
    """What :func:`residual_norm` gives: the residual stream behind the block, its norm for
    the next block, and the statistics that :func:`residual_norm_grad` takes (float32, per
    row the mean and reciprocal deviation of ``residual``, then those of the block where it
    has a norm)."""

    residual: torch.Tensor
    out: torch.Tensor
    stats: torch.Tensor


class ResidualNormGrads(NamedTuple):
    """The gradients of :func:`residual_norm`'s operands; ``None`` for those it had not."""

    residual: torch.Tensor
    block: Optional[torch.Tensor]
    weight: torch.Tensor
    bias: Optional[torch.Tensor]
    block_weight: Optional[torch.Tensor]
    block_bias: Optional[torch.Tensor]
    gate: Optional[torch.Tensor]


def _kind(kind: str) -> int:
    try:
        return KINDS[kind]
    except KeyError:
        raise ValueError(f"unknown norm {kind!r}; expected one of {sorted(KINDS)}") from None


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, residual, block, weight, bias, block_weight, block_bias, gate, scale, eps, kind):
        following, out, stats = _native.norm(residual, block, weight, bias, block_weight, block_bias,
                                             gate, scale, eps, kind)
        ctx.save_for_backward(residual if block is None else following, stats, block, weight, bias,
                              block_weight, block_bias, gate)
        ctx.scale, ctx.kind = scale, kind
        ctx.mark_non_differentiable(stats)
        ctx.set_materialize_grads(False)
        return following, out, stats

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_residual, grad_out, _):
        if grad_residual is None and grad_out is None:
            return (None,) * 10
        following, stats, block, weight, bias, block_weight, block_bias, gate = ctx.saved_tensors
        grads = _native.norm_grad(grad_out, grad_residual, following, stats, block, weight, bias,
                                  block_weight, block_bias, gate, ctx.scale, ctx.kind)
        return (*(g if need else None for g, need in zip(grads, ctx.needs_input_grad)), None, None,
                None)


def _norm(residual, block, weight, bias, block_weight, block_bias, gate, scale, eps, kind):
    args = (residual, block, weight, bias, block_weight, block_bias, gate)
    if torch.is_autocast_enabled():
        args = of_one_type(args, torch.float32)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args):
        return _ResidualNorm.apply(*args, scale, eps, _kind(kind))
    return _native.norm(*args, scale, eps, _kind(kind))


def norm(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
         eps: float = 1e-5, kind: str = "rms") -> torch.Tensor:
    """``norm(x) * weight + bias`` over the last dimension.

    ``kind`` is ``"rms"`` (``x / sqrt(mean(x ** 2) + eps)``) or ``"layer"`` (the same of ``x``
    without its mean, with an optional ``bias``).  Rows have 1 to 16384 values of float32 / float16 /
    bfloat16, at any stride; weights are ``[width]``, of the same type (under ``torch.autocast``
    operands of several types are cast to float32, in which torch's norms run there).  Differences from
    the mean and their squares are taken in 32 bits; a row where they pass these comes out as
    zeros or NaN.  For the norms at a model's beginning; :func:`residual_norm` is the norm behind a
    residual sum.
    """
    return _norm(x, None, weight, bias, None, None, None, 1.0, eps, kind)[1]


def residual_norm(residual: torch.Tensor, block: torch.Tensor, weight: torch.Tensor,
                  bias: Optional[torch.Tensor] = None,
                  block_weight: Optional[torch.Tensor] = None,
                  block_bias: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                  scale: float = 1.0, eps: float = 1e-5, kind: str = "rms") -> ResidualNorm:
    """What lies between two blocks of a model, in one pass.

    ``block`` is the output of a block that read the residual stream ``residual`` (both
    ``[..., width]``).  With ``u = norm(block) * block_weight + block_bias`` (``block``
    itself without ``block_weight``), the results are ``residual + scale * gate * u`` and its
    ``norm * weight + bias``, which the next block reads.  ``gate`` is ``[width]``, or as
    ``residual`` with a size of 1 in the last of its leading dimensions (``[batch, 1, width]``:
    one for each sequence; ``[batch, time, width]``: for each token).  ``kind``, ``eps``, types and
    sizes are those of :func:`norm`, for both norms; biases go with ``"layer"``.

    Computed in 32 bits, each result rounded once; ``out`` comes from the sum before it is
    rounded.  All operands are differentiable; the backward pass keeps the new residual and
    the block's output, no normalised copies.
    """
    return ResidualNorm(*_norm(residual, block, weight, bias, block_weight, block_bias, gate, scale,
                               eps, kind))


def residual_norm_grad(grad_out: Optional[torch.Tensor], grad_residual: Optional[torch.Tensor],
                       residual: torch.Tensor, stats: torch.Tensor, block: torch.Tensor,
                       weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                       block_weight: Optional[torch.Tensor] = None,
                       block_bias: Optional[torch.Tensor] = None,
                       gate: Optional[torch.Tensor] = None, scale: float = 1.0,
                       kind: str = "rms") -> ResidualNormGrads:
    """The gradients of :func:`residual_norm`'s operands.

    ``residual`` and ``stats`` are its results (the residual stream *behind* the block), the other
    operands its own; ``grad_out`` or ``grad_residual`` may be ``None`` (zeros).  Sums over
    rows are made in 32 bits in an order that follows from the sizes, and rounded once.
    """
    return ResidualNormGrads(*_native.norm_grad(grad_out, grad_residual, residual, stats, block,
                                                weight, bias, block_weight, block_bias, gate, scale,
                                                _kind(kind)))
