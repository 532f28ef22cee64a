"""The gradient of a bias beside a frozen weight, captured and replayed: every replay gives the sum of its inputs.

A sum of T terms takes at most T additions, each off by 2^-24 of the sum of magnitudes; half a step of the type written besides."""
from __future__ import annotations

import pytest
import torch
from act8_oracle import DTYPES, ROUND
from side_stream import side_stream

from stagehand_amd.act8 import linear_act8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,out", [(1, 8), (300, 40), (16384, 64), (100000, 8), (4099, 1155)])
def test_a_bias_beside_a_frozen_weight(tokens, out, dtype):
    x, w = torch.randn(tokens, 32, device="cuda", dtype=dtype), torch.randn(out, 32, device="cuda", dtype=dtype)
    b = torch.randn(out, device="cuda", dtype=dtype, requires_grad=True)
    dy = torch.randn(tokens, out, device="cuda", dtype=dtype)

    def step():
        return torch.autograd.grad(linear_act8(x, w, b), (b,), dy)[0]

    side = side_stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        db = step()
    for _ in range(4):
        dy.normal_()
        graph.replay()
        torch.cuda.synchronize()
        want, size = dy.double().sum(0), dy.double().abs().sum(0)
        for got in (db, step()):
            assert bool(((got.double() - want).abs() <= tokens * 2.0 ** -24 * size + ROUND[dtype] * want.abs()).all())
