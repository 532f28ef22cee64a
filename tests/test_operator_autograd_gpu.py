"""What the operators do not differentiate, or overwrite, autograd hears of: it raises where it would otherwise
give wrong gradients."""
from __future__ import annotations

import pytest
import torch

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

