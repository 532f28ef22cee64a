"""The example's block: norms, adapters and recomputation on kept activations together, as they are used.

A kept value is off by at most 2^k / 2 with 2^k <= 2 max / 127, max the largest of its 32 neighbours: 2^k / sqrt(12) <= max /
220 in the mean, and the largest of 32 values is at most some 3.5 of their standard deviations: 1.6%. The gradients are
linear in each of the kept activations that they are made from, of which a path through the block has three at most: 5%.
"""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch
from side_stream import side_stream

from stagehand_amd.act8 import quantize_activation

pytestmark = pytest.mark.gpu

SPEC = importlib.util.spec_from_file_location("lora_block_act8", Path(__file__).resolve().parent.parent / "examples" / "lora_block_act8.py")
example = importlib.util.module_from_spec(SPEC)
SPEC.loader.exec_module(example)


def make(dtype, tokens=200, hidden=256, heads=4, rank=8):
    block = example.Block(hidden, heads, rank, dtype)
    g = torch.Generator(device="cuda").manual_seed(1)
    x, dy = (torch.randn(2, tokens, hidden, device="cuda", generator=g).to(dtype) for _ in range(2))
    return block, x, torch.randn(2, hidden, device="cuda", generator=g).to(dtype), dy


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradients_are_near_those_of_kept_tensors(dtype):
    block, x, vec, dy = make(dtype)
    for recompute in (False, True):
        _, got = example.step(block, x, vec, dy, True, recompute)
        _, want = example.step(block, x, vec, dy, False, recompute)
        assert len(got) == 9
        for p, q in zip(got, want):
            assert p.shape == q.shape and bool(p.isfinite().all())
            assert float((p.float() - q.float()).norm()) <= 0.05 * float(q.float().norm())


def test_recomputation_is_that_of_the_kept_input():
    block, x, vec, dy = make(torch.bfloat16)
    _, got = example.step(block, x, vec, dy, True, True)
    at = quantize_activation(x).dequantize()
    _, want = example.step(block, at, vec, dy, True, False)
    for p, q in zip(got[1:], want[1:]):
        assert torch.equal(p, q)


def test_what_is_kept():
    """Recomputed: the block's input in 8.25 bits. Else: the norms' inputs, the adapters' inputs and outputs in less than the
    tensors take."""
    block, x, vec, dy = make(torch.bfloat16, tokens=2048)
    example.step(block, x, vec, dy, True)  # what libraries allocate once
    kept = {(k, r): example.step(block, x, vec, dy, k, r)[0] for k in (True, False) for r in (True, False)}
    assert kept[True, True] <= 1.04 * x.numel() + (1 << 18) < 2 * x.numel() <= kept[False, True]
    assert kept[True, False] < kept[False, False]


def test_a_captured_step_replays():
    block, x, vec, dy = make(torch.bfloat16)
    leaf = x.clone().requires_grad_()
    params = block.adapters()

    def run():
        return torch.autograd.grad(block(leaf, vec, True), (leaf, *params), dy)

    side = side_stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for n in range(3):
        with torch.no_grad():
            leaf.copy_(x * (1 + n))
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(outs, run()):
            assert float((p.float() - q.float()).norm()) <= 0.01 * float(q.float().norm())  # attention's gradient has no fixed order
