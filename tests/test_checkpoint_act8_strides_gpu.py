"""A function is recomputed from an input that lies in memory as the input of its first call did."""
from __future__ import annotations

import pytest
import torch
from torch.nn import functional as F

from stagehand_amd.act8 import checkpoint_act8, quantize_activation

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("needs_grad", [True, False])
def test_views_that_only_the_inputs_order_allows(needs_grad):
    """Heads before tokens in shape, behind them in memory, as attention leaves them."""
    w = torch.randn(48, 96, device="cuda", requires_grad=True)
    memory = torch.randn(2, 10, 3, 32, device="cuda")
    x = memory.transpose(1, 2).requires_grad_(needs_grad)

    def project(t):
        return F.linear(torch.sin(t).transpose(1, 2).view(2, 10, 96), w)

    dy = torch.randn(2, 10, 48, device="cuda")
    inputs = (x, w) if needs_grad else (w,)
    got = torch.autograd.grad(checkpoint_act8(project, x), inputs, dy)
    at = quantize_activation(memory).dequantize().transpose(1, 2).requires_grad_(needs_grad)
    want = torch.autograd.grad(project(at), (at, w) if needs_grad else (w,), dy)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_strides_of_the_recomputations_input():
    base = torch.randn(4, 6, 64, device="cuda")
    # dense tensors keep their order; of others, and of expanded ones, the order is all that can be kept
    for x, strides in ((base, (384, 64, 1)), (base.transpose(0, 1), (64, 384, 1)), (base.permute(2, 0, 1), (1, 384, 64)), (base[0, 0], (1,)),
                       (base[:, ::2], (192, 64, 1)), (base[..., 3:40].transpose(0, 1), (37, 222, 1)), (base[:1].expand(4, 6, 64), None)):
        seen = []

        def f(t):
            seen.append((t.shape, t.stride()))
            return t.sin()

        x = x.detach().requires_grad_()
        dx, = torch.autograd.grad(checkpoint_act8(f, x).sum(), (x,))
        at = quantize_activation(x.detach()).dequantize()
        assert torch.equal(dx, at.cos())
        assert len(seen) == 2 and seen[0] == (x.shape, x.stride()) and seen[1][0] == x.shape
        if strides is not None:
            assert seen[1][1] == strides
