"""Weight gradients from fp32 gradients near the least numbers of the type.

The matrix cores get three bf16 parts of a gradient, and bf16's least number is 2^-133: parts of a gradient from 2^-110 on lose
none of its 24 bits, below that what lies under 2^-133 is cut. So a weight's gradient is off by at most 2^-133 of the sum of the
kept inputs' magnitudes, besides the roundings of its sum; a bias' gradient is summed from the gradients as they are.
"""
from __future__ import annotations

import act8_oracle as oracle
import pytest
import torch
from act8_oracle import activations
from test_weight_grad_act8_gpu import close, products

from stagehand_amd.act8 import quantize_activation, weight_grad_act8

pytestmark = pytest.mark.gpu

SIZES = [(1, 8, 32), (40, 33, 70), (300, 130, 200), (4096, 32, 256)]


def gradients(tokens, out, low, high):
    """Of magnitudes from 2^low on, below 2^high, with random bits."""
    g = torch.Generator(device="cuda").manual_seed(tokens)
    size = torch.exp2(torch.randint(low, high, (tokens, out), device="cuda", generator=g).double())
    v = size * (1 + torch.rand(tokens, out, device="cuda", generator=g, dtype=torch.float64))
    return torch.where(torch.rand(tokens, out, device="cuda", generator=g) < 0.5, v, -v).float()


@pytest.mark.parametrize("low,high,cut", [(-110, -100, 0.0), (-116, -114, 2.0 ** -133), (-127, -120, 2.0 ** -133), (-149, -126, 2.0 ** -133)])
@pytest.mark.parametrize("tokens,out,inp", SIZES)
def test_small_gradients(tokens, out, inp, low, high, cut):
    dy = gradients(tokens, out, low, high)
    x = activations(tokens, inp, seed=tokens) * 2.0 ** 60  # so that the sums are ordinary numbers
    dw, db = weight_grad_act8(dy, quantize_activation(x), bias=True)
    kept = oracle.kept_values(x)
    want, size, want_b, size_b = products(dy, kept)
    lost = cut * kept.abs().sum(0).cuda()
    err = ((dw.double() - want).abs() - lost).clamp_min(0)
    bad = err > (tokens + 32) * 2.0 ** -23 * size + 2.0 ** -24 * want.abs()
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float(err.max())}"
    close(db, want_b, size_b, tokens, "dbias")
