"""Log probabilities of given tokens, with entropy and top alternatives."""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _native


class TokenLogprobs(NamedTuple):
    """What :func:`token_logprobs` gives, per row of logits, in float32."""

    logprob: torch.Tensor
    entropy: Optional[torch.Tensor]
    lse: torch.Tensor
    top_logprob: Optional[torch.Tensor]
    top_id: Optional[torch.Tensor]


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top, entropy, ignore_index):
        logprob, ent, lse, top_logprob, top_id = _native.token_logprobs(logits, targets, top,
                                                                        entropy, ignore_index)
        ctx.save_for_backward(logits, targets, lse, ent)
        ctx.ignore_index = ignore_index
        ctx.mark_non_differentiable(*(t for t in (lse, top_logprob, top_id) if t is not None))
        ctx.set_materialize_grads(False)
        return logprob, ent, lse, top_logprob, top_id

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_logprob, grad_entropy, *_):
        logits, targets, lse, ent = ctx.saved_tensors
        if grad_logprob is None and grad_entropy is None:
            return None, None, None, None, None
        return _native.token_logprobs_grad(logits, targets, lse, grad_logprob, ent, grad_entropy,
                                           ctx.ignore_index), None, None, None, None


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, top: int = 0,
                   entropy: bool = False, ignore_index: int = -100) -> TokenLogprobs:
    """Log probabilities of ``targets`` under ``softmax(logits)``.

    ``logits`` is ``[..., vocab]`` (float32 / float16 / bfloat16, rows at any
    stride), ``targets`` ``[...]`` (int64 or int32).  One pass over the logits
    gives, per row: ``logprob`` of the target (0 where the target is
    ``ignore_index``), ``lse`` (the log of the sum of exponentials), with
    ``entropy=True`` the entropy of the distribution, and with ``top=k`` (up to
    64) the ``k`` likeliest tokens as ``top_logprob`` and ``top_id``, in falling
    order, equal ones by rising index.  ``logprob`` and ``entropy`` are
    differentiable, so that ``-token_logprobs(logits, targets).logprob.mean()`` is
    a cross-entropy loss.  ``lse`` and the alternatives are not: a loss on them adds
    nothing to the gradients.  (``logits.gather(-1, targets[..., None])[..., 0] - logprob``
    is an ``lse`` that has a gradient.)

    A row that a mask left nothing (all ``-inf``) has log probability ``-inf``,
    entropy 0 and a gradient of zeros.  A row with NaN or ``+inf`` gives NaN, and
    so does a target outside the vocabulary.
    """
    if logits.requires_grad and torch.is_grad_enabled():
        return TokenLogprobs(*_TokenLogprobs.apply(logits, targets, top, entropy, ignore_index))
    return TokenLogprobs(*_native.token_logprobs(logits, targets, top, entropy, ignore_index))


def token_logprobs_grad(logits: torch.Tensor, targets: torch.Tensor, lse: torch.Tensor,
                        grad_logprob: Optional[torch.Tensor],
                        entropy: Optional[torch.Tensor] = None,
                        grad_entropy: Optional[torch.Tensor] = None,
                        ignore_index: int = -100) -> torch.Tensor:
    """The gradient of the logits of :func:`token_logprobs`.

    With ``p = softmax(logits)``: ``grad_logprob * (onehot(target) - p) -
    grad_entropy * p * (log p + entropy)``, rounded once to the logits' type.
    ``lse`` and ``entropy`` are the forward pass's; the row gradients are float32.
    """
    return _native.token_logprobs_grad(logits, targets, lse, grad_logprob, entropy, grad_entropy,
                                       ignore_index)
