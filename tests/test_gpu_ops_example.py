"""The operators in a training loop with the engine: the example GPT.

The model learns one fixed batch.  Its first loss is the plain model's (the same
forward values in fp32, up to the order of sums); along the way the activations'
8 bits, with an error of at most 1/127 of their block's largest value, may not
change what it learns."""

from __future__ import annotations

import math

import pytest
import torch

import minispeed_amd as ms
from minispeed_amd.examples import train_lm

pytestmark = pytest.mark.gpu
SIZES = dict(vocab=301, block=64, d=64, layers=2, heads=2)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_the_example_learns_as_the_plain_model_does(dtype):
    ours = train_lm.train(dtype, 60, micro=4, **SIZES)
    plain = train_lm.train(dtype, 60, micro=4, plain=True, **SIZES)
    assert abs(ours[0] - math.log(301)) < 0.1
    assert abs(ours[0] - plain[0]) <= (1e-5 if dtype == "fp32" else 2e-2)
    assert ours[-1] < 0.6 * ours[0]
    assert abs(ours[-1] - plain[-1]) < 0.1 * plain[0]


def test_an_overflow_in_a_held_activation_skips_the_step():
    """An inf in an activation that only exists in 8 bits reaches the gradients as
    NaN; the engine skips the step and halves the loss scale."""
    torch.manual_seed(0)
    model = train_lm.GPT(**SIZES).to("cuda")
    config = {"train_micro_batch_size_per_gpu": 2, "gradient_accumulation_steps": 1, "dtype": "fp16",
              "fp16": {"enabled": True, "loss_scale": 0, "initial_scale_power": 8},
              "optimizer": {"type": "AdamW", "params": {"lr": 1e-3}},
              "zero_optimization": {"stage": 1}, "steps_per_print": 10 ** 9}
    engine, _, _, _ = ms.initialize(model=model, model_parameters=model.parameters(), config=config)
    h = torch.randn(8, 64, device="cuda", dtype=torch.float16)
    block = model.blocks[0]
    hidden = block.fc(h)
    hidden.data[3, 5] = float("-inf")
    scale = engine.get_loss_scale()
    before = engine.flat_groups[0].data.clone()
    y = ms.ops.activation8_linear(hidden, block.fc2.weight, block.fc2.bias, "silu")
    engine.backward(y.nan_to_num(0.0, 0.0, 0.0).float().mean())
    assert engine.step() is False
    assert engine.get_loss_scale() == scale / 2
    assert torch.equal(engine.flat_groups[0].data, before)


def test_the_command_runs(capsys):
    assert train_lm.main(["--dtype", "bf16", "--steps", "3"]) == 0
    out = capsys.readouterr().out
    assert "step    0" in out and "entropy" in out
