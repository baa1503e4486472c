"""Forward and backward pass of the block and head operators through autograd, captured into one
graph and replayed with new inputs, on another stream's memory between the replays; two graphs
of the same operator replayed in turn."""

from __future__ import annotations

import pytest
import torch

import minispeed_amd as ms

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _step(kind, leaves, extra):
    if kind == "linear":
        r = ms.ops.linear_logprobs(leaves[0], leaves[1], extra[0])
        outs = [r.logprob, r.lse]
    elif kind == "norm":
        r = ms.ops.residual_norm(*leaves[:2], leaves[2], leaves[3], leaves[4], None, leaves[5],
                                 scale=0.5, kind="layer")
        outs = [r.residual, r.out]
    else:
        outs = [ms.ops.position_bias(leaves[0], 50, 70, causal=False)]
    return [*(o.detach() for o in outs),
            *torch.autograd.grad(outs, leaves, grad_outputs=extra[-len(outs):])]


def _inputs(kind, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    if kind == "linear":
        return ([randn(150, 64).half(), (randn(700, 64) * 0.1).half()],
                [torch.randint(0, 700, (150,), generator=g, device=DEV), randn(150), randn(150)])
    if kind == "norm":
        rows = [randn(4, 30, 264).bfloat16() for _ in range(2)]
        return ([*rows, *(randn(264).bfloat16() for _ in range(3)), randn(4, 1, 264).bfloat16()],
                [randn(4, 30, 264).bfloat16() for _ in range(2)])
    return [randn(32, 4)], [randn(4, 50, 70)]


@pytest.mark.parametrize("kind", ["linear", "norm", "bias"])
def test_captured_and_replayed(kind):
    def capture(seed):
        leaves, extra = _inputs(kind, seed)
        leaves = [t.requires_grad_() for t in leaves]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _step(kind, leaves, extra)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _step(kind, leaves, extra)
        return graph, leaves, extra, out

    graphs = [capture(1), capture(2)]
    for seed in range(3, 7):
        for graph, leaves, extra, out in graphs:
            new_leaves, new_extra = _inputs(kind, seed)
            with torch.no_grad():
                for a, b in zip((*leaves, *extra), (*new_leaves, *new_extra)):
                    a.copy_(b)
            torch.full((1 << 22,), float("nan"), device=DEV)
            graph.replay()
            torch.cuda.synchronize()
            want = _step(kind, [t.requires_grad_() for t in new_leaves], new_extra)
            assert all(torch.equal(a, b) for a, b in zip(out, want)), (kind, seed)


@pytest.mark.parametrize("kind", ["linear", "norm", "bias"])
def test_two_streams_at_once(kind):
    sets = [_inputs(kind, seed) for seed in (11, 12)]
    wants = [_step(kind, [t.requires_grad_() for t in leaves], extra) for leaves, extra in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    outs = [[], []]
    for _ in range(6):
        for k, (leaves, extra) in enumerate(sets):
            with torch.cuda.stream(streams[k]):
                outs[k].append(_step(kind, leaves, extra))
    torch.cuda.synchronize()
    for out, want in zip(outs, wants):
        for again in out:
            assert all(torch.equal(a, b) for a, b in zip(again, want))
