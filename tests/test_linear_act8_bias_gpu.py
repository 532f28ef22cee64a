"""The bias of a Linear that keeps its input in 8 bits learns by itself, whatever the input's dims."""
from __future__ import annotations

import pytest
import torch

from stagehand_amd.act8 import linear_act8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(64,), (1, 64), (5, 64), (2, 3, 64), (0, 64)])
@pytest.mark.parametrize("out", [1, 8])
def test_a_bias_beside_a_frozen_weight(shape, out):
    x, w = torch.randn(shape, device="cuda"), torch.randn(out, 64, device="cuda")
    b = torch.randn(out, device="cuda", requires_grad=True)
    dy = torch.randn(*shape[:-1], out, device="cuda")
    db, = torch.autograd.grad(linear_act8(x, w, b), (b,), dy)
    rows = dy.double().view(-1, out)
    assert db.shape == b.shape
    # six terms at most: five additions, each off by 2^-24 of the sum of magnitudes
    assert bool(((db.double() - rows.sum(0)).abs() <= 5 * 2.0 ** -24 * rows.abs().sum(0)).all())
