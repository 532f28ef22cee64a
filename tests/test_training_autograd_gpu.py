"""What the training operators do not differentiate, or overwrite, autograd hears of."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from stagehand_amd.act8 import checkpoint_act8, linear_act8, quantize_activation, weight_grad_act8
from stagehand_amd.layer_norm import layer_norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("grad_mode", [True, False])
def test_tangents_are_refused(grad_mode):
    x, w, b, dy = (torch.randn(s, device="cuda") for s in ((4, 64), (64,), (64,), (4, 8)))
    a = torch.randn(8, 64, device="cuda")
    kept = quantize_activation(x)
    with torch.set_grad_enabled(grad_mode), forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        calls = [lambda: layer_norm(dual(x), w, b), lambda: layer_norm(x, dual(w), b), lambda: layer_norm(x, w, dual(b)),
                 lambda: layer_norm(x, out=dual(torch.zeros_like(x))), lambda: quantize_activation(dual(x)),
                 lambda: kept.dequantize(out=dual(torch.zeros_like(x))), lambda: weight_grad_act8(dual(dy), kept),
                 lambda: linear_act8(dual(x), a), lambda: linear_act8(x, dual(a))]
        if grad_mode:
            calls.append(lambda: checkpoint_act8(torch.sin, dual(x)))
        for i, call in enumerate(calls):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
                pytest.fail(f"call {i} was not refused")
        layer_norm(x, w, b)  # nothing that has a tangent: as always


def test_transforms_of_torch_func_are_refused():
    x, a = torch.randn(4, 64, device="cuda"), torch.randn(8, 64, device="cuda")
    for f in (lambda t: layer_norm(t), lambda t: linear_act8(t, a)):
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, (x,), (torch.ones_like(x),))
        with pytest.raises(RuntimeError):
            torch.func.vmap(f)(torch.stack((x, x)))
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda t: f(t).sum())(x)


def test_gradients_add_up_over_uses():
    """One norm's weight for two inputs, one input for two norms, and a broadcast scale."""
    x, w, b = torch.randn(2, 9, 96, device="cuda", requires_grad=True), torch.randn(96, device="cuda", requires_grad=True), torch.randn(96, device="cuda")
    c = torch.randn(2, 9, 96, device="cuda")
    total = torch.autograd.grad((layer_norm(x, w, b) + layer_norm(2 * x, w)), (x, w), c)
    one, two = torch.autograd.grad(layer_norm(x, w, b), (x, w), c), torch.autograd.grad(layer_norm(2 * x, w), (x, w), c)
    for t, p, q in zip(total, one, two):  # each is rounded once, their sum once more
        assert bool(((t - p - q).abs() <= 2.0 ** -23 * (p.abs() + q.abs())).all())
    scale = torch.randn(1, 1, 96, device="cuda", requires_grad=True)
    wide = torch.autograd.grad(layer_norm(x, scale.expand(2, 1, 96), modulate=True), (scale,), c)[0]
    shared = torch.autograd.grad(layer_norm(x, scale, modulate=True), (scale,), c)[0]
    size = (c * layer_norm(x)).abs().sum((0, 1), keepdim=True)
    assert wide.shape == shared.shape == scale.shape
    assert bool(((wide - shared).abs() <= 2.0 ** -24 * 80 * size).all())  # 18 terms in another order, at 40 roundings each


def test_backward_twice_and_after_an_overwritten_input():
    for keep8 in (False, True):
        x = torch.randn(5, 300, device="cuda", requires_grad=True)
        h = x * 1
        y = layer_norm(h, keep8=keep8)
        c = torch.randn_like(y)
        first = torch.autograd.grad(y, x, c, retain_graph=True)[0]
        assert torch.equal(first, torch.autograd.grad(y, x, c, retain_graph=True)[0])
        with torch.no_grad():
            h.add_(1)
        if keep8:  # the kept input is the norm's own
            assert torch.equal(first, torch.autograd.grad(y, x, c)[0])
        else:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                torch.autograd.grad(y, x, c)
    x, w = torch.randn(5, 64, device="cuda"), torch.randn(8, 64, device="cuda", requires_grad=True)
    y = checkpoint_act8(lambda t: torch.sin(t) @ w.t(), x)
    c = torch.randn_like(y)
    first = torch.autograd.grad(y, w, c, retain_graph=True)[0]
    assert torch.equal(first, torch.autograd.grad(y, w, c)[0])


def test_layers_without_tokens():
    w, b = torch.randn(8, 64, device="cuda", requires_grad=True), torch.randn(8, device="cuda", requires_grad=True)
    x = torch.empty(0, 3, 64, device="cuda", requires_grad=True)
    dx, dw, db = torch.autograd.grad(linear_act8(x, w, b), (x, w, b), torch.empty(0, 3, 8, device="cuda"))
    assert dx.shape == x.shape and not dw.any() and not db.any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens, out", [(5, 33), (40, 1), (77, 1155), (1013, 301), (300, 64)])
def test_gradients_expanded_over_tokens(dtype, tokens, out):
    """A sum over the tokens sends back one row for all of them: the same gradients as from a copy of it for each."""
    x = torch.randn(tokens, 96, device="cuda", dtype=dtype)
    w, b = (torch.randn(s, device="cuda", dtype=dtype, requires_grad=True) for s in ((out, 96), (out,)))
    row = torch.randn(out, device="cuda", dtype=dtype)
    y = linear_act8(x, w, b)
    got = torch.autograd.grad(y.sum(0), (w, b), row, retain_graph=True)
    want = torch.autograd.grad(y, (w, b), row.expand(tokens, out).contiguous())
    for g, e in zip(got, want):
        assert torch.equal(g, e)
    dy = row.expand(tokens, out)
    for g, e in zip(weight_grad_act8(dy, quantize_activation(x), bias=True), want):
        assert torch.equal(g, e)


def test_layers_without_outputs():
    for shape in ((64,), (5, 64), (2, 3, 64), (0, 64)):
        x = torch.randn(shape, device="cuda", requires_grad=True)
        w, b = torch.empty(0, 64, device="cuda", requires_grad=True), torch.empty(0, device="cuda", requires_grad=True)
        y = linear_act8(x, w, b)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
        assert dx.shape == x.shape and not dx.any() and dw.shape == w.shape and db.shape == b.shape
