"""Train a small GPT with the language-model operators and the engine together.

    python -m minispeed_amd.examples.train_lm [--dtype fp16] [--steps 40] [--fused]

A decoder of the layout of minispeed's examples/train_lm.py:62-115 in which

* the token table is read by ``ms.ops.embedding`` and its gradient summed in token
  order, the same bits on every run;
* each attention half-block runs under ``ms.ops.checkpoint8``: its input is held
  in 8 bits and the half-block computed again in the backward pass;
* each MLP's second product is ``ms.ops.activation8_linear``, which keeps the hidden
  layer in 8 bits for the activation's and the weight's gradients;
* the loss is the mean of ``-ms.ops.token_logprobs``, which also reports the entropy
  of the predictions.

``plain=True`` builds the same model from torch's own operations.

``fused=True`` (``--fused``) is a decoder of the same sizes whose residual stream is touched
only between its half-blocks: ``ms.ops.norm`` and ``ms.ops.residual_norm`` (a norm behind each
half-block, a gate for each channel, the residual sum and the norm before the next), with
positions from ``ms.ops.position_bias`` in the attention mask instead of a table, and
the loss from ``ms.ops.linear_logprobs``, which never stores the logits, with a small
penalty on their normaliser.  ``plain=True`` beside it is again torch's operations.
"""

from __future__ import annotations

import argparse
import math

import torch
import torch.nn.functional as F
from torch import nn

import minispeed_amd as ms


class Block(nn.Module):
    def __init__(self, d: int, heads: int, plain: bool):
        super().__init__()
        self.heads, self.plain = heads, plain
        self.ln1, self.qkv, self.proj = nn.LayerNorm(d), nn.Linear(d, 3 * d), nn.Linear(d, d)
        self.ln2, self.fc, self.fc2 = nn.LayerNorm(d), nn.Linear(d, 4 * d), nn.Linear(4 * d, d)

    def attend(self, x):
        b, t, c = x.shape
        q, k, v = (z.view(b, t, self.heads, -1).transpose(1, 2).float()
                   for z in self.qkv(self.ln1(x)).chunk(3, dim=-1))
        att = F.scaled_dot_product_attention(q, k, v, is_causal=True)
        return self.proj(att.to(x.dtype).transpose(1, 2).reshape(b, t, c))

    def forward(self, x):
        if self.plain:
            x = x + self.attend(x)
            return x + self.fc2(F.gelu(self.fc(self.ln2(x))))
        x = x + ms.ops.checkpoint8(self.attend, x)
        return x + ms.ops.activation8_linear(self.fc(self.ln2(x)), self.fc2.weight, self.fc2.bias)


class GPT(nn.Module):
    """Returns the mean loss of ``idx``'s next tokens and their mean entropy."""

    def __init__(self, vocab=512, block=128, d=256, layers=4, heads=4, plain=False):
        super().__init__()
        self.plain, self.block = plain, block
        self.wte, self.wpe = nn.Embedding(vocab, d), nn.Embedding(block, d)
        self.blocks = nn.ModuleList(Block(d, heads, plain) for _ in range(layers))
        self.ln_f = nn.LayerNorm(d)
        with torch.no_grad():
            for p in self.parameters():
                if p.dim() > 1:
                    p.normal_(0.0, 0.02)

    def forward(self, idx):
        inputs, targets = idx[:, :-1], idx[:, 1:]
        if self.plain:
            x = self.wte(inputs)
        else:
            x = ms.ops.embedding(inputs, self.wte.weight)
        x = x + self.wpe.weight[:inputs.shape[1]]
        for blk in self.blocks:
            x = blk(x)
        logits = F.linear(self.ln_f(x), self.wte.weight)
        if self.plain:
            logp = F.log_softmax(logits.float(), -1)
            entropy = -(logp.exp() * logp).sum(-1)
            return -logp.gather(-1, targets[..., None]).mean(), entropy.mean().detach()
        r = ms.ops.token_logprobs(logits, targets, entropy=True)
        return -r.logprob.mean(), r.entropy.mean().detach()


class FusedBlock(nn.Module):
    """A block's parameters: of the norm before each half-block, those inside, and of the norm and
    gate behind each."""

    def __init__(self, d: int, heads: int):
        super().__init__()
        self.heads = heads
        self.ln1, self.qkv, self.proj = nn.LayerNorm(d), nn.Linear(d, 3 * d), nn.Linear(d, d)
        self.ln2, self.fc, self.fc2 = nn.LayerNorm(d), nn.Linear(d, 4 * d), nn.Linear(4 * d, d)
        self.post1, self.post2 = nn.LayerNorm(d), nn.LayerNorm(d)
        self.gate1, self.gate2 = (nn.Parameter(torch.full((d,), 0.3)) for _ in range(2))

    def attend(self, y, mask):
        b, t, c = y.shape
        q, k, v = (z.view(b, t, self.heads, -1).transpose(1, 2).float()
                   for z in self.qkv(y).chunk(3, dim=-1))
        att = F.scaled_dot_product_attention(q, k, v, attn_mask=mask.float())
        return self.proj(att.to(y.dtype).transpose(1, 2).reshape(b, t, c))


class FusedGPT(nn.Module):
    """Returns the mean loss of ``idx``'s next tokens and their mean ``lse``."""

    def __init__(self, vocab=512, block=128, d=256, layers=4, heads=4, plain=False, buckets=32,
                 max_distance=64, penalty=1e-4):
        super().__init__()
        self.plain, self.max_distance, self.penalty, self.block = plain, max_distance, penalty, block
        self.wte, self.positions = nn.Embedding(vocab, d), nn.Parameter(torch.zeros(buckets, heads))
        self.blocks = nn.ModuleList(FusedBlock(d, heads) for _ in range(layers))
        self.ln_f = nn.LayerNorm(d)
        with torch.no_grad():
            for p in self.parameters():
                if p.dim() > 1:
                    p.normal_(0.0, 0.02)

    def _mask(self, t):
        if not self.plain:
            return ms.ops.position_bias(self.positions, t, t, max_distance=self.max_distance,
                                        causal=True)
        n = self.positions.shape[0]
        away = torch.arange(t, device="cuda")[:, None] - torch.arange(t, device="cuda")[None, :]
        ratio = torch.log(away.clamp(min=1).double() * 2 / n) / math.log(2 * self.max_distance / n)
        wide = (n // 2 + (ratio * (n - n // 2) + 1e-9).floor().long()).clamp(max=n - 1)
        bucket = torch.where(away < n // 2, away.clamp(min=0), wide)
        return self.positions[bucket].permute(2, 0, 1).masked_fill(away < 0, -math.inf)

    def _between(self, x, out, post, gate, following):
        """What lies between a half-block and the next: (residual, its norm)."""
        if self.plain:
            u = F.layer_norm(out.float(), (out.shape[-1],), post.weight.float(), post.bias.float())
            x = (x.float() + gate.float() * u).to(x.dtype)
            return x, following(x)
        r = ms.ops.residual_norm(x, out, following.weight, following.bias, post.weight, post.bias, gate,
                                 kind="layer")
        return r.residual, r.out

    def forward(self, idx):
        inputs, targets = idx[:, :-1], idx[:, 1:]
        x = self.wte(inputs) if self.plain else ms.ops.embedding(inputs, self.wte.weight)
        mask = self._mask(inputs.shape[1])
        first = self.blocks[0].ln1 if len(self.blocks) else self.ln_f
        y = first(x) if self.plain else ms.ops.norm(x, first.weight, first.bias, kind="layer")
        for k, blk in enumerate(self.blocks):
            x, y = self._between(x, blk.attend(y, mask), blk.post1, blk.gate1, blk.ln2)
            h = blk.fc(y)
            out = (blk.fc2(F.gelu(h)) if self.plain
                   else ms.ops.activation8_linear(h, blk.fc2.weight, blk.fc2.bias))
            last = k + 1 == len(self.blocks)
            x, y = self._between(x, out, blk.post2, blk.gate2, self.ln_f if last else self.blocks[k + 1].ln1)
        if self.plain:
            logits = F.linear(y, self.wte.weight).float()
            lse = torch.logsumexp(logits, -1)
            logprob = logits.gather(-1, targets[..., None])[..., 0] - lse
        else:
            logprob, lse = ms.ops.linear_logprobs(y, self.wte.weight, targets)
        return -logprob.mean() + self.penalty * (lse ** 2).mean(), lse.mean().detach()


def train(dtype: str = "fp16", steps: int = 40, micro: int = 8, seed: int = 0, plain: bool = False,
          verbose: bool = False, fused: bool = False, **sizes):
    """The losses of ``steps`` boundaries on one fixed batch of random tokens."""
    torch.manual_seed(seed)
    model = (FusedGPT if fused else GPT)(plain=plain, **sizes).to("cuda")
    config = {"train_micro_batch_size_per_gpu": micro, "gradient_accumulation_steps": 1,
              "gradient_clipping": 1.0, "dtype": dtype,
              "fp16": {"enabled": dtype == "fp16", "loss_scale": 0, "initial_scale_power": 12},
              "optimizer": {"type": "AdamW", "params": {"lr": 1e-3, "weight_decay": 0.01}},
              "zero_optimization": {"stage": 1}, "steps_per_print": 10 ** 9}
    engine, _, _, _ = ms.initialize(model=model, model_parameters=model.parameters(),
                                    config=config)
    vocab, block = model.wte.num_embeddings, model.block
    gen = torch.Generator().manual_seed(seed + 1)
    idx = torch.randint(0, vocab, (micro, block + 1), generator=gen).to("cuda")
    losses = []
    for step in range(steps):
        loss, mean = engine(idx)
        engine.backward(loss)
        engine.step()
        losses.append(float(loss.detach()))
        if verbose and (step % 10 == 0 or step == steps - 1):
            print(f"step {step:4d}  loss {losses[-1]:.4f}  {'lse' if fused else 'entropy'} {float(mean):.4f}  "
                  f"grad norm {engine.grad_norm:.3f}", flush=True)
    return losses


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description="Train a small GPT on one batch of random tokens.")
    ap.add_argument("--dtype", choices=("fp32", "fp16", "bf16"), default="fp16")
    ap.add_argument("--steps", type=int, default=40)
    ap.add_argument("--fused", action="store_true",
                    help="norms, gates and residual sums in one pass, the loss without logits")
    ap.add_argument("--plain", action="store_true", help="torch's operations instead")
    args = ap.parse_args(argv)
    train(args.dtype, args.steps, plain=args.plain, verbose=True, fused=args.fused)
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
