"""Log probabilities of given tokens straight from hidden states and the head's weight."""

from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import _native
from ._types import of_one_type


class LinearLogprobs(NamedTuple):
    """What :func:`linear_logprobs` gives, per row of hidden states, in float32."""

    logprob: torch.Tensor
    lse: torch.Tensor


class _LinearLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, targets, scale, ignore_index):
        logprob, lse = _native.linear_logprobs(hidden, weight, targets, scale, ignore_index)
        ctx.save_for_backward(hidden, weight, targets, lse)
        ctx.scale, ctx.ignore_index = scale, ignore_index
        ctx.set_materialize_grads(False)
        return logprob, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_logprob, grad_lse):
        hidden, weight, targets, lse = ctx.saved_tensors
        need = ctx.needs_input_grad
        if (grad_logprob is None and grad_lse is None) or not (need[0] or need[1]):
            return None, None, None, None, None
        dh, dw = _native.linear_logprobs_grad(hidden, weight, targets, lse, grad_logprob, grad_lse,
                                              ctx.scale, ctx.ignore_index, need[0], need[1])
        return dh, dw, None, None, None


def linear_logprobs(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor,
                    scale: float = 1.0, ignore_index: int = -100) -> LinearLogprobs:
    """Log probabilities of ``targets`` under ``softmax(scale * hidden @ weight.T)``.

    ``hidden`` is ``[..., width]``, ``weight`` ``[vocab, width]``, of one type (float32 /
    float16 / bfloat16), ``targets`` ``[...]`` (int64 or int32).  The logits are not stored,
    forward or backward.  Beside the operands and the gradients a call takes some
    bytes for each token and 128 words of the vocabulary.  Backward takes

    * the gradients of a piece of the logits, in the operands' type: 512 MiB at most, or 256 words'
      worth of the vocabulary;
    * sums in 32 bits: of ``hidden``'s gradient where the vocabulary is gone through in several
      pieces (4 bytes for each value), and of products that are cut into parts: 128 MiB of these at
      most, but up to 1.25 GiB for float32 operands and where one gradient is wanted alone;
    * a copy of ``hidden`` in float16, if the weight's gradient is wanted.

    Both take copies of 2-byte operands whose rows are not on 16-byte boundaries, and of
    float32 ones of many tokens always (6 bytes for each value).

    Per row: ``logprob`` of the target (0 where it is ``ignore_index``, NaN where it is outside
    the vocabulary) and ``lse``, the log of the sum of exponentials.  Both are
    differentiable: ``-r.logprob.mean() + z * (r.lse ** 2).mean()`` is a cross entropy with a
    penalty on the normaliser.  Gradients are rounded once to the operands' type, from sums in
    32 bits over terms of that type.  Rows without a gradient add nothing to ``weight``'s
    unless they hold infinities or NaN themselves.

    Under ``torch.autocast``, operands of two types are cast to autocast's, as a product's are.
    """
    if torch.is_autocast_enabled():
        hidden, weight = of_one_type((hidden, weight))
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
        return LinearLogprobs(*_LinearLogprobs.apply(hidden, weight, targets, scale, ignore_index))
    return LinearLogprobs(*_native.linear_logprobs(hidden, weight, targets, scale, ignore_index))


def linear_logprobs_grad(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor,
                         lse: torch.Tensor, grad_logprob: Optional[torch.Tensor],
                         grad_lse: Optional[torch.Tensor] = None, scale: float = 1.0,
                         ignore_index: int = -100) -> Tuple[torch.Tensor, torch.Tensor]:
    """The gradients of ``hidden`` and ``weight`` of :func:`linear_logprobs`.

    With ``p = softmax(scale * hidden @ weight.T)`` and ``d = grad_logprob * (onehot(target) -
    p) + grad_lse * p``: ``scale * d @ weight`` and ``scale * d.T @ hidden``.  ``lse`` is
    the forward pass's; the row gradients are float32.
    """
    return _native.linear_logprobs_grad(hidden, weight, targets, lse, grad_logprob, grad_lse, scale,
                                        ignore_index, True, True)
