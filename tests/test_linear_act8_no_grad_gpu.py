"""A Linear that keeps its input in 8 bits keeps nothing where nothing will be differentiated."""
from __future__ import annotations

import pytest
import torch
from torch.nn import functional as F

from stagehand_amd import act8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_nothing_is_kept_without_gradients(monkeypatch, mode):
    x = torch.randn(3, 50, 64, device="cuda", requires_grad=True)
    w, b = torch.randn(40, 64, device="cuda", requires_grad=True), torch.randn(40, device="cuda", requires_grad=True)
    kept = act8.quantize_activation(x.detach())

    def unexpected(*args, **kw):
        raise AssertionError("the input was quantised")

    monkeypatch.setattr(act8, "quantize_activation", unexpected)
    with mode():
        want = F.linear(x, w, b)
        for given in (None, kept):
            before = torch.cuda.memory_allocated()
            y = act8.linear_act8(x, w, b, given)
            assert torch.cuda.memory_allocated() - before <= -(-y.numel() * y.element_size() // 512) * 512
            assert torch.equal(y, want) and not y.requires_grad
        with torch.autocast("cuda", dtype=torch.bfloat16):
            assert torch.equal(act8.linear_act8(x, w, b), F.linear(x, w, b))
        # an input that could not be kept
        assert act8.linear_act8(x[..., :0], w[:, :0], b).shape == y.shape
        with pytest.raises(ValueError):  # arguments are checked all the same
            act8.linear_act8(x, w[:, :63], b)
    with pytest.raises(AssertionError, match="quantised"):
        act8.linear_act8(x, w, b)


def test_the_first_pass_of_a_reentrant_checkpoint_keeps_nothing(monkeypatch):
    from torch.utils.checkpoint import checkpoint

    x, w = torch.randn(5, 64, device="cuda", requires_grad=True), torch.randn(8, 64, device="cuda", requires_grad=True)
    calls, quantize = [], act8.quantize_activation
    monkeypatch.setattr(act8, "quantize_activation", lambda t: calls.append(1) or quantize(t))
    y = checkpoint(lambda t: act8.linear_act8(t, w), x, use_reentrant=True)
    assert not calls
    y.sum().backward()
    assert len(calls) == 1 and w.grad is not None
