"""What the operators do not differentiate, or overwrite, autograd hears of: it raises where it would otherwise
give wrong gradients."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from stagehand_amd.int8 import Int8Weight, linear_i8, matmul_i8, quantize_tokens
from stagehand_amd.qk_norm import qk_norm_rope

pytestmark = pytest.mark.gpu


def weight(out=64, inp=96):
    g = torch.Generator().manual_seed(0)
    return Int8Weight(torch.randint(-128, 128, (out, inp), dtype=torch.int8, generator=g).cuda(), torch.rand(out, device="cuda"))


def heads(*shape):
    return torch.randn(shape, device="cuda", dtype=torch.bfloat16)


# ── out= is a write that autograd sees ───────────────────────────────────────


@pytest.mark.parametrize("which", ["linear_i8", "matmul_i8"])
@pytest.mark.parametrize("tokens", [3, 200])
def test_a_saved_tensor_that_the_product_overwrites_makes_backward_raise(tokens, which):
    w, x = weight(), torch.randn(tokens, 96, device="cuda")
    a = torch.ones(tokens, 64, device="cuda", requires_grad=True)
    wide = torch.randn(tokens, 200, device="cuda")
    out = wide[:, 8:72]
    y = a * out  # saves out for the gradient of a
    before = out._version
    with torch.no_grad():
        linear_i8(x, w, out=out) if which == "linear_i8" else matmul_i8(quantize_tokens(x), w, out=out)
    assert out._version > before and wide._version == out._version and x._version == 0
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_saved_heads_that_the_norms_overwrite_make_backward_raise():
    for view in (False, True):
        base = heads(2, 9, 6, 32)
        q, k = base[:, :, :4].transpose(1, 2), base[:, :, 4:].transpose(1, 2)
        a = torch.ones_like(base if view else q).requires_grad_()
        y = a * (base if view else q)
        qk_norm_rope(q, k, out=(q, k))
        assert base._version >= 2
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


def test_only_outputs_change_their_version():
    q, k, w = heads(1, 2, 5, 32), heads(1, 2, 5, 32), torch.ones(32, device="cuda", dtype=torch.bfloat16)
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    qk_norm_rope(q, k, w, w, out=(qo, ko))
    qk_norm_rope(q, None, w, out=(qo, None))
    assert (qo._version, ko._version) == (2, 1) and not (q._version or k._version or w._version)
    with torch.inference_mode():  # tensors without versions are written all the same
        fresh = torch.empty_like(q)
        qk_norm_rope(q, None, out=(fresh, None))
        x = torch.randn(3, 96, device="cuda")
        linear_i8(x, weight(), out=torch.empty(3, 64, device="cuda"))


# ── out= that requires a gradient ────────────────────────────────────────────


def test_out_that_requires_grad_is_refused():
    w, x = weight(), torch.randn(4, 96, device="cuda")
    out = torch.zeros(4, 64, device="cuda", requires_grad=True)
    q, k = heads(1, 2, 5, 32), heads(1, 2, 5, 32)
    qo, ko = torch.zeros_like(q).requires_grad_(), torch.zeros_like(k)
    calls = [lambda: linear_i8(x, w, out=out), lambda: matmul_i8(quantize_tokens(x), w, out=out),
             lambda: linear_i8(x, w, out=(out * 1)), lambda: qk_norm_rope(q, k, out=(qo, ko)),
             lambda: qk_norm_rope(q, k, out=(ko, qo))]
    for call in calls:
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
    assert not out.any() and not qo.any() and not ko.any()
    with torch.no_grad():  # as any in-place operation
        assert torch.equal(linear_i8(x, w, out=out), linear_i8(x, w))
        assert torch.equal(qk_norm_rope(q, k, out=(qo, ko))[0], qk_norm_rope(q, k)[0])


# ── forward-mode derivatives ─────────────────────────────────────────────────


@pytest.mark.parametrize("grad_mode", [True, False])
def test_tangents_are_refused(grad_mode):
    w, x = weight(), torch.randn(4, 96, device="cuda")
    q, k = heads(1, 2, 5, 32).float(), heads(1, 2, 5, 32).float()
    n, cos = torch.ones(32, device="cuda"), torch.ones(5, 16, device="cuda")
    with torch.set_grad_enabled(grad_mode), forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        calls = [lambda: linear_i8(dual(x), w), lambda: quantize_tokens(dual(x)),
                 lambda: matmul_i8(quantize_tokens(x)._replace(scale=dual(torch.ones(4, device="cuda"))), w),
                 lambda: linear_i8(x, w, out=dual(torch.zeros(4, 64, device="cuda"))),
                 lambda: qk_norm_rope(dual(q), k, n, n, cos, cos), lambda: qk_norm_rope(q, dual(k), n, n, cos, cos),
                 lambda: qk_norm_rope(q, k, dual(n), n, cos, cos), lambda: qk_norm_rope(q, k, n, dual(n), cos, cos),
                 lambda: qk_norm_rope(q, k, n, n, dual(cos), cos), lambda: qk_norm_rope(q, k, n, n, cos, dual(cos)),
                 lambda: qk_norm_rope(q, None, out=(dual(torch.zeros_like(q)), None))]
        if grad_mode:
            calls.append(lambda: qk_norm_rope(dual(q), k, n.clone().requires_grad_(), n, cos, cos))
        for i, call in enumerate(calls):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
                pytest.fail(f"call {i} was not refused")
        # nothing that has a tangent: as always
        assert torch.equal(linear_i8(x, w), matmul_i8(quantize_tokens(x), w, out_dtype=torch.float32))
        qk_norm_rope(q, k, n, n, cos, cos)


def test_transforms_of_torch_func_are_refused():
    w, x, q = weight(), torch.randn(4, 96, device="cuda"), heads(1, 2, 5, 32).float()
    for f, at in ((lambda t: linear_i8(t, w), x), (lambda t: qk_norm_rope(t, None)[0], q)):
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, (at,), (torch.ones_like(at),))
        with pytest.raises(RuntimeError):
            torch.func.vmap(f)(torch.stack((at, at)))
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda t: f(t).sum())(at)


def test_token_scales_that_require_grad_are_refused():
    t = quantize_tokens(torch.randn(4, 96, device="cuda"))
    t = t._replace(scale=t.scale.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="no gradient"):
        matmul_i8(t, weight())
    with torch.no_grad():
        matmul_i8(t, weight())
