"""The block and head operators together, as the example's fused model uses them: its gradients
against those of the same model from torch's operations, and its run in the engine.

Tolerances: in fp32 the two models differ by the order of sums (2^-24 each, some thousand terms and
a dozen layers deep: 2e-5 of a gradient's norm) and by the activations that are held in 8 bits for
the gradients (half a step of 1/127 of a block's largest value: below 1% of a gradient's
norm, in every parameter that a held value reaches, which is all of them before the last
product)."""

from __future__ import annotations

import math

import pytest
import torch

import minispeed_amd as ms
from minispeed_amd.examples import train_lm

pytestmark = pytest.mark.gpu
SIZES = dict(vocab=301, block=64, d=64, layers=2, heads=2)


def _grads(plain, dtype, **more):
    torch.manual_seed(0)
    model = train_lm.FusedGPT(plain=plain, **SIZES, **more).to("cuda", dtype)
    gen = torch.Generator().manual_seed(1)
    idx = torch.randint(0, 301, (3, 65), generator=gen).to("cuda")
    with torch.no_grad():
        model.positions.normal_(0.0, 0.5)
    loss, lse = model(idx)
    loss.backward()
    return loss.detach(), lse, {k: p.grad for k, p in model.named_parameters()}


def test_gradients_are_those_of_the_plain_model():
    ours, plain = _grads(False, torch.float32, penalty=0.01), _grads(True, torch.float32, penalty=0.01)
    assert abs(float(ours[0] - plain[0])) <= 1e-5 * float(plain[0])
    assert abs(float(ours[1] - plain[1])) <= 1e-5 * float(plain[1])
    for name, want in plain[2].items():
        got = ours[2][name]
        assert got is not None and got.shape == want.shape, name
        assert float((got - want).norm()) <= 0.01 * float(want.norm()) + 1e-7, name


def test_gradients_without_the_8_bit_activations(monkeypatch):
    """The three operators alone: with the activation's own gradients in the place of the held
    ones, the models agree to the order of their sums."""
    monkeypatch.setattr(ms.ops, "activation8_linear",
                        lambda h, w, b: torch.nn.functional.linear(torch.nn.functional.gelu(h), w, b))
    ours, plain = _grads(False, torch.float32, penalty=0.01), _grads(True, torch.float32, penalty=0.01)
    for name, want in plain[2].items():
        assert float((ours[2][name] - want).norm()) <= 2e-5 * float(want.norm()) + 1e-8, name


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_it_runs_in_the_engine(dtype):
    losses = train_lm.train(dtype, 4, micro=2, fused=True, **SIZES)
    assert len(losses) == 4 and all(math.isfinite(x) for x in losses)
    assert abs(losses[0] - math.log(301)) < 0.2


def test_the_command_runs(capsys):
    assert train_lm.main(["--dtype", "bf16", "--steps", "3", "--fused"]) == 0
    assert "lse" in capsys.readouterr().out
