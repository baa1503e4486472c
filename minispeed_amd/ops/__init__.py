"""Operators of a language model's training step, as HIP kernels for gfx950.

* :func:`embedding`, :func:`embedding_grad` — the scaled token embedding and its
  gradient, summed in token order (the same bits on every run);
* :func:`token_logprobs`, :func:`token_logprobs_grad` — the log probability of a
  given token per position, with entropy and the most likely alternatives, and
  the gradient of the logits;
* :func:`pack8`, :func:`unpack8`, :func:`checkpoint8`, :func:`activation8`,
  :func:`activation8_grad`, :func:`activation8_linear` — activations held in 8
  bits between forward and backward.

``embedding``, ``token_logprobs``, ``activation8``, ``checkpoint8`` and
``activation8_linear`` take part in autograd; the ``_grad`` functions are the same backward
passes for a program that calls them itself, and are not differentiable again.  Forward-mode derivatives are refused.  All of them
run on the current stream, allocate through torch's caching allocator and return before
the kernels have finished.
"""

from .activation8 import (Checkpoint8, activation8, activation8_grad, activation8_linear,
                          checkpoint8, pack8, unpack8)
from .embedding import embedding, embedding_grad
from .logprobs import TokenLogprobs, token_logprobs, token_logprobs_grad

__all__ = [
    "Checkpoint8",
    "TokenLogprobs",
    "activation8",
    "activation8_grad",
    "activation8_linear",
    "checkpoint8",
    "embedding",
    "embedding_grad",
    "pack8",
    "token_logprobs",
    "token_logprobs_grad",
    "unpack8",
]
