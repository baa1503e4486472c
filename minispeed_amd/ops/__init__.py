"""Operators of a language model's training step, as HIP kernels for gfx950.

* :func:`embedding`, :func:`embedding_grad` — the scaled token embedding and its
  gradient, summed in token order (the same bits on every run);
* :func:`token_logprobs`, :func:`token_logprobs_grad` — the log probability of a
  given token per position, with entropy and the most likely alternatives, and
  the gradient of the logits;
* :func:`linear_logprobs`, :func:`linear_logprobs_grad` — the same log probability straight
  from the hidden states and the head's weight, without storing the logits, and both
  gradients;
* :func:`norm`, :func:`residual_norm`, :func:`residual_norm_grad` — the norms before and
  after a block with its gate, residual scale and residual sum, and all their gradients;
* :func:`position_bias`, :func:`position_bias_grad` — the learned relative position bias of
  attention by buckets of distances, and its table's gradient;
* :func:`pack8`, :func:`unpack8`, :func:`checkpoint8`, :func:`activation8`,
  :func:`activation8_grad`, :func:`activation8_linear` — activations held in 8
  bits between forward and backward.

``embedding``, ``token_logprobs``, ``linear_logprobs``, ``norm``, ``residual_norm``,
``position_bias``, ``activation8``, ``checkpoint8`` and ``activation8_linear`` take part in autograd; the ``_grad`` functions are the same backward
passes for a program that calls them itself, and are not differentiable again.  Forward-mode derivatives are refused.  All of them
run on the current stream, allocate through torch's caching allocator and return before
the kernels have finished.
"""

from .activation8 import (Checkpoint8, activation8, activation8_grad, activation8_linear,
                          checkpoint8, pack8, unpack8)
from .embedding import embedding, embedding_grad
from .linear import LinearLogprobs, linear_logprobs, linear_logprobs_grad
from .logprobs import TokenLogprobs, token_logprobs, token_logprobs_grad
from .norm import (ResidualNorm, ResidualNormGrads, norm, residual_norm, residual_norm_grad)
from .posbias import position_bias, position_bias_grad

__all__ = [
    "Checkpoint8",
    "LinearLogprobs",
    "ResidualNorm",
    "ResidualNormGrads",
    "TokenLogprobs",
    "activation8",
    "activation8_grad",
    "activation8_linear",
    "checkpoint8",
    "embedding",
    "embedding_grad",
    "linear_logprobs",
    "linear_logprobs_grad",
    "norm",
    "pack8",
    "position_bias",
    "position_bias_grad",
    "residual_norm",
    "residual_norm_grad",
    "token_logprobs",
    "token_logprobs_grad",
    "unpack8",
]
