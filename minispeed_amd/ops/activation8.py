"""Activations held in 8 bits between forward and backward.

Blocks of 32 consecutive values share a power-of-two scale of one byte; a value
is a signed byte times that scale, 1.03 bytes in all.  The error of a value is
at most half a step, less than 1/127 of its block's largest magnitude.  A block
that holds an inf or a NaN comes back as NaN throughout, so that an overflow in
a held activation still reaches the gradients and the loss scaler skips the
step.
"""

from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch
import torch.nn.functional as F
from torch.utils._pytree import tree_leaves

from . import _native

KINDS = {"gelu": 0, "gelu_tanh": 1, "silu": 2, "swiglu": 3}


class Checkpoint8:
    """A tensor in its 8-bit form: ``codes`` (int8, one per value), ``exponents``
    (uint8, one per 32 values), and the ``shape`` and ``dtype`` it comes back
    with."""

    __slots__ = ("codes", "exponents", "shape", "dtype")

    def __init__(self, codes: torch.Tensor, exponents: torch.Tensor, shape, dtype: torch.dtype):
        self.codes, self.exponents = codes, exponents
        self.shape, self.dtype = tuple(shape), dtype

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.exponents.numel()


def pack8(x: torch.Tensor) -> Checkpoint8:
    """The 8-bit form of ``x`` (float32 / float16 / bfloat16).  Its whole numbers carry no
    gradient, and neither does what :func:`unpack8` makes of them."""
    codes, exponents = _native.pack8(x)
    return Checkpoint8(codes, exponents, x.shape, x.dtype)


def unpack8(held: Checkpoint8) -> torch.Tensor:
    """The values that an 8-bit form stands for."""
    return _native.unpack8(held.codes, held.exponents, held.shape, held.dtype)


def _kind(kind: str) -> int:
    try:
        return KINDS[kind]
    except KeyError:
        raise ValueError(f"unknown activation {kind!r}; expected one of {sorted(KINDS)}") from None


class _Activation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, up, kind):
        a, *held = _native.act8(h, up, _kind(kind))
        ctx.kind, ctx.meta, ctx.gated = kind, (h.shape, h.dtype), up is not None
        ctx.save_for_backward(*held)
        ctx.mark_non_differentiable(*(t for t in held if t is not None))
        ctx.set_materialize_grads(False)
        return a, *held

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, *_):
        if grad is None:
            return None, None, None
        held = ctx.saved_tensors
        saved = [Checkpoint8(held[k], held[k + 1], *ctx.meta) for k in ((0, 2) if ctx.gated else (0,))]
        grads, _ = activation8_grad(saved, grad, ctx.kind, again=False)
        return grads[0], grads[1] if ctx.gated else None, None


def activation8(h: torch.Tensor, kind: str = "gelu", up: Optional[torch.Tensor] = None
                ) -> Tuple[torch.Tensor, Tuple[Checkpoint8, ...]]:
    """``(a, saved)``: the activation of ``h`` and its input in 8 bits, in one pass.

    ``kind`` is ``"gelu"`` (with the error function), ``"gelu_tanh"``, ``"silu"`` or
    ``"swiglu"`` (``silu(h) * up``).  ``a`` is computed from ``h`` itself; ``saved``
    (one checkpoint, two for ``"swiglu"``) is what :func:`activation8_grad` takes.  ``a``
    is differentiable, by the held values.
    """
    if torch.is_grad_enabled() and (h.requires_grad or (up is not None and up.requires_grad)):
        a, codes, exponents, up_codes, up_exponents = _Activation.apply(h, up, kind)
    else:
        a, codes, exponents, up_codes, up_exponents = _native.act8(h, up, _kind(kind))
    saved = (Checkpoint8(codes, exponents, h.shape, h.dtype),)
    if up is not None:
        saved += (Checkpoint8(up_codes, up_exponents, h.shape, h.dtype),)
    return a, saved


def activation8_grad(saved: Sequence[Checkpoint8], grad: torch.Tensor, kind: str = "gelu",
                     again: bool = True
                     ) -> Tuple[Tuple[torch.Tensor, ...], Optional[torch.Tensor]]:
    """``(grads, a)``: the backward pass of :func:`activation8`, in one pass.

    ``grads`` holds the gradient of ``h`` (and of ``up``); ``a`` is the activation
    again, from the held values, for the weight gradient of the product behind it
    (``None`` with ``again=False``).
    """
    if not 1 <= len(saved) <= 2:
        raise ValueError(f"{len(saved)} checkpoints, expected one or two")
    for s in saved:
        if s.dtype != grad.dtype or s.shape != tuple(grad.shape):
            raise ValueError(f"grad is {grad.dtype} {tuple(grad.shape)}, the checkpoint "
                             f"{s.dtype} {s.shape}")
    up = saved[1] if len(saved) == 2 else None
    dh, dup, a = _native.act8_grad(saved[0].codes, saved[0].exponents, up and up.codes,
                                   up and up.exponents, grad, _kind(kind), again)
    return ((dh,) if dup is None else (dh, dup)), a


class _ActivationLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, up, weight, bias, kind):
        a, saved = activation8(h, kind, up)
        ctx.kind, ctx.meta = kind, [(s.shape, s.dtype) for s in saved]
        ctx.save_for_backward(weight, *(t for s in saved for t in (s.codes, s.exponents)))
        ctx.bias_dtype = None if bias is None else bias.dtype
        return F.linear(a, weight, bias)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        weight, *held = ctx.saved_tensors
        saved = [Checkpoint8(held[2 * k], held[2 * k + 1], *m) for k, m in enumerate(ctx.meta)]
        need = ctx.needs_input_grad
        dh = dup = dw = db = None
        flat = grad.reshape(-1, grad.shape[-1])
        if need[0] or need[1] or need[2]:
            if need[0] or need[1]:
                # (the types differ under autocast only)
                da = grad.matmul(weight.to(grad.dtype)).to(saved[0].dtype)
            else:
                # only the activation again is used, on which these values have no bearing
                da = torch.empty(saved[0].shape, dtype=saved[0].dtype, device=grad.device)
            grads, a = activation8_grad(saved, da, ctx.kind, again=need[2])
            dh, dup = grads if len(grads) == 2 else (grads[0], None)
            if need[2]:
                dw = flat.t().mm(a.reshape(-1, a.shape[-1]).to(grad.dtype)).to(weight.dtype)
        if ctx.bias_dtype is not None and need[3]:
            db = flat.sum(0, dtype=ctx.bias_dtype)
        return dh, dup, dw, db, None


def activation8_linear(h: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                       kind: str = "gelu", up: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``linear(act(h), weight, bias)`` that keeps only ``h`` (and ``up``) in 8 bits.

    The second half of a transformer's MLP.  torch would keep ``h`` for the
    activation and ``act(h)`` for the weight's gradient, 4 bytes per value in half
    precision; this keeps 1.03 (2.06 gated).  The backward pass reads the held
    values once, for the gradient of ``h`` and for the activation that the weight's
    gradient needs.  The products are the library's.
    """
    return _ActivationLinear.apply(h, up, weight, bias, kind)


class _Checkpoint(torch.autograd.Function):
    @staticmethod
    def forward(ctx, fn, preserve_rng, *args):
        ctx.fn, ctx.preserve_rng = fn, preserve_rng
        ctx.autocast = dict(device_type="cuda", enabled=torch.is_autocast_enabled("cuda"),
                            dtype=torch.get_autocast_dtype("cuda"))
        if preserve_rng:
            ctx.rng = _rng_state(args)
        ctx.slots, held = [], []
        for arg in args:
            if not isinstance(arg, torch.Tensor):
                ctx.slots.append(("value", arg, False))
            elif _is_activation(arg):
                packed = pack8(arg)
                ctx.slots.append(("held", (packed.shape, packed.dtype), arg.requires_grad))
                held += [packed.codes, packed.exponents]
            else:
                ctx.slots.append(("tensor", None, arg.requires_grad))
                held.append(arg)
        ctx.save_for_backward(*held)
        with torch.no_grad():
            out = fn(*args)
        for o in out if isinstance(out, tuple) else (out,):
            # autograd would not see tensors in it
            if not isinstance(o, torch.Tensor) and any(isinstance(t, torch.Tensor)
                                                       for t in tree_leaves(o)):
                raise TypeError(f"fn gives a {type(o).__name__}; expected a tensor or a tuple "
                                "of tensors")
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        held, args = list(ctx.saved_tensors), []
        for what, meta, needs in ctx.slots:
            if what == "value":
                arg = meta
            elif what == "held":
                codes, exponents = held.pop(0), held.pop(0)
                arg = unpack8(Checkpoint8(codes, exponents, *meta))
            else:
                arg = held.pop(0).detach()
            if needs:
                arg.requires_grad_()
            args.append(arg)
        with torch.enable_grad(), torch.autocast(**ctx.autocast), \
                _RngOf(ctx.rng if ctx.preserve_rng else None):
            out = ctx.fn(*args)
        outs = out if isinstance(out, tuple) else (out,)
        pairs = [(o, g) for o, g in zip(outs, grads)
                 if isinstance(o, torch.Tensor) and o.requires_grad and g is not None]
        if pairs:
            torch.autograd.backward([o for o, _ in pairs], [g for _, g in pairs])
        return None, None, *(a.grad if needs else None
                             for a, (_, _, needs) in zip(args, ctx.slots))


_HELD = (torch.float32, torch.float16, torch.bfloat16)


def _is_activation(arg):
    """What is held in 8 bits: gradients flow through it, to something that is no parameter."""
    return (arg.is_cuda and arg.dim() > 0 and arg.dtype in _HELD and arg.requires_grad
            and not isinstance(arg, torch.nn.Parameter))


def _rng_state(args):
    device = next((a.device for a in args if isinstance(a, torch.Tensor) and a.is_cuda), None)
    return (torch.get_rng_state(), device,
            None if device is None else torch.cuda.get_rng_state(device))


class _RngOf:
    """Inside, the random generators are where ``state`` was taken; afterwards they
    are where they were."""

    def __init__(self, state):
        self.state = state

    def __enter__(self):
        if self.state is not None:
            device = self.state[1]
            self.now = (torch.get_rng_state(), device,
                        None if device is None else torch.cuda.get_rng_state(device))
            self._set(self.state)

    def __exit__(self, *exc):
        if self.state is not None:
            self._set(self.now)

    @staticmethod
    def _set(state):
        cpu, device, cuda = state
        torch.set_rng_state(cpu)
        if device is not None:
            torch.cuda.set_rng_state(cuda, device)


def checkpoint8(fn, *args, preserve_rng_state: bool = True):
    """``fn(*args)`` whose activations are computed again in the backward pass, from
    arguments held in 8 bits.

    The float32, float16 and bfloat16 tensors on the GPU among ``args`` that require a
    gradient are kept in their 8-bit form, and ``fn`` runs again on the values
    they stand for when the gradients come: the use of minispeed's ``checkpoint``
    (minispeed/activation_checkpointing.py:17-20) with a quarter to a half of its
    memory.  Parameters, which are there anyway, and tensors without a gradient (masks,
    whose infinities no 8-bit form has, and tables) are kept as they are.  The first run
    sees the arguments themselves.  ``fn`` gives a tensor or a tuple of them (and of
    other things, which are passed on).  Parameters that ``fn``
    reaches by itself get their gradients; with ``preserve_rng_state`` random
    operations (dropout) draw the same numbers in both runs.  If none of ``args``
    requires a gradient there is nothing to hold, and ``fn`` runs as it would by itself.
    """
    if not torch.is_grad_enabled() or not any(isinstance(a, torch.Tensor) and a.requires_grad
                                              for a in args):
        return fn(*args)
    return _Checkpoint.apply(fn, preserve_rng_state, *args)
