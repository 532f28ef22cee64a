"""Weight gradients from kept inputs, and the layers and recomputation that keep them, against products in 64 bits.

Tolerance: the factors are exact (three bf16 parts hold the 24 bits of a float32), so are the products of 8 by 8 or 11
by 7 bits in float32. A sum of T of them takes at most T additions, in whatever order and joined from however many parts;
if each rounded in the worst way it would be off by 2^-23 of the sum of magnitudes: (T + 32) 2^-23 of that, which covers the 3 T
additions of parts too (the smaller parts add 2^-8 of the first), plus half a step of the type written.
"""
from __future__ import annotations

import act8_oracle as oracle
import pytest
import torch
from act8_oracle import DTYPES, ROUND, TINY, activations
from side_stream import side_stream
from torch.nn import functional as F

from stagehand_amd.act8 import checkpoint_act8, linear_act8, quantize_activation, weight_grad_act8

pytestmark = pytest.mark.gpu

SIZES = [  # tokens, out, in
    (1, 1, 1), (1, 8, 32), (2, 7, 31), (31, 32, 33), (32, 33, 64), (33, 64, 65), (77, 65, 257), (128, 16, 1155), (129, 256, 256),
    (1013, 40, 500), (200, 1000, 1155), (4096, 32, 1024), (300, 257, 129), (70, 3000, 2100), (520, 4100, 4130), (300, 1900, 1899),
    (8000, 1001, 1155), (900, 257, 300),
]


def products(dy, kept_values):
    """(dweight, its sum of magnitudes, dbias, its) in 64 bits on the device."""
    d, x = dy.reshape(-1, dy.shape[-1]).double(), kept_values.cuda()
    dt, at = d.t().contiguous(), d.abs().t().contiguous()
    return dt @ x, at @ x.abs(), d.sum(0), d.abs().sum(0)


def close(got, want, size, terms, what):
    dt = got.dtype
    want = want.double()
    err = (got.double() - want).abs()
    bad = ~(err <= (terms + 32) * 2.0 ** -23 * size + ROUND[dt] * want.abs() + TINY[dt])
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(err.max())}"


def check(dy, x, dw, db=None):
    want, size, want_b, size_b = products(dy, oracle.kept_values(x.reshape(-1, x.shape[-1])))
    terms = max(1, dy.numel() // max(1, dy.shape[-1]))
    close(dw, want, size, terms, "dweight")
    if db is not None:
        close(db, want_b, size_b, terms, "dbias")


def make(tokens, out, inp, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    return (0.1 * torch.randn(tokens, out, device="cuda", generator=g)).to(dtype), activations(tokens, inp, dtype=dtype, seed=seed)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,out,inp", SIZES)
def test_matches_64_bits(tokens, out, inp, dtype):
    dy, x = make(tokens, out, inp, dtype, seed=tokens)
    kept = quantize_activation(x)
    dw, db = weight_grad_act8(dy, kept, bias=True)
    assert dw.dtype == db.dtype == dtype and dw.shape == (out, inp) and db.shape == (out,)
    check(dy, x, dw, db)
    alone, none = weight_grad_act8(dy, kept)
    assert none is None and torch.equal(alone, dw)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("out_dtype", DTYPES)
def test_types_of_the_result(dtype, out_dtype):
    for tokens, out, inp in ((700, 24, 100), (40, 130, 70)):
        dy, x = make(tokens, out, inp, dtype)
        dw, db = weight_grad_act8(dy, quantize_activation(x), bias=True, out_dtype=out_dtype)
        assert dw.dtype == db.dtype == out_dtype
        check(dy, x, dw, db)


@pytest.mark.parametrize("dtype", DTYPES)
def test_views_and_leading_dims(dtype):
    base, x = make(4 * 33, 300, 100, dtype)
    base, x = base.view(4, 33, 300), x.view(4, 33, 100)
    kept = quantize_activation(x)
    for dy in (base[..., 5:86], base[..., :64], base[..., 7:], base[..., ::2], base[:, :, 299:], base[:, :1].expand(4, 33, 300)):
        check(dy, x, *weight_grad_act8(dy, kept, bias=True))
    short = quantize_activation(x[:, ::2])
    check(base[:, ::2, 3:70], x[:, ::2], *weight_grad_act8(base[:, ::2, 3:70], short, bias=True))
    one = quantize_activation(x[0, 0])
    check(base[0, 0], x[0, 0], *weight_grad_act8(base[0, 0], one, bias=True))


@pytest.mark.parametrize("dtype", DTYPES)
def test_ends_of_the_range(dtype):
    """Large and small factors, fp16's subnormals among them, lose nothing on the way."""
    info = torch.finfo(dtype)
    tokens, out, inp = 64, 40, 96
    dy, x = make(tokens, out, inp, torch.float32)
    low = 2.0 ** -14 if dtype == torch.float16 else 2.0 ** -60
    x[:, :32] *= low / 8
    x[:, 32:64] = x[:, 32:64] / x[:, 32:64].abs().max() * min(info.max, 2.0 ** 60)
    dy[:, ::2] *= low
    dy, x = dy.to(dtype), x.to(dtype)
    dw, db = weight_grad_act8(dy, quantize_activation(x), bias=True, out_dtype=torch.float32)
    check(dy, x, dw, db)


@pytest.mark.parametrize("dtype", DTYPES)
def test_broken_values_stay_their_own(dtype):
    for tokens, out, inp in ((100, 24, 100), (70, 200, 300), (1000, 40, 70)):
        dy, x = make(tokens, out, inp, dtype)
        x[3, 40] = float("nan")
        x[tokens - 1, 66] = float("inf")
        dy[7, 5], dy[9, out - 1] = float("inf"), float("nan")
        dw, db = weight_grad_act8(dy, quantize_activation(x), bias=True)
        broken = torch.zeros(out, inp, dtype=torch.bool)
        broken[:, 32:96] = True  # the groups of both
        broken[5], broken[out - 1] = True, True
        assert bool(dw[~broken.cuda()].isfinite().all())
        assert bool(dw[:, 32:64].isnan().all()) and bool(dw[:, 64:min(96, inp)].isnan().all()) and bool(dw[out - 1].isnan().all())
        assert bool((~dw[5].isfinite()).all()) and float(db[5]) == float("inf") and bool(db[-1].isnan())
        clean_x, clean_dy = x.clone(), dy.clone()
        clean_x[3, 40] = clean_x[tokens - 1, 66] = 0
        clean_dy[7, 5] = clean_dy[9, out - 1] = 0
        same, _ = weight_grad_act8(clean_dy, quantize_activation(clean_x))
        assert torch.equal(dw[~broken.cuda()], same[~broken.cuda()])


def test_no_tokens_and_no_outputs():
    for dtype in DTYPES:
        kept = quantize_activation(torch.empty(0, 70, device="cuda", dtype=dtype))
        dw, db = weight_grad_act8(torch.empty(0, 33, device="cuda", dtype=dtype), kept, bias=True)
        assert dw.shape == (33, 70) and not dw.any() and not db.any()
        kept = quantize_activation(torch.ones(5, 70, device="cuda", dtype=dtype))
        assert weight_grad_act8(torch.empty(5, 0, device="cuda", dtype=dtype), kept)[0].shape == (0, 70)


def test_repeated_calls_give_the_same_bits():
    for tokens, out, inp in ((4096, 32, 1024), (500, 500, 500), (2000, 128, 256)):
        dy, x = make(tokens, out, inp, torch.bfloat16)
        kept = quantize_activation(x)
        first = weight_grad_act8(dy, kept, bias=True)
        for _ in range(3):
            again = weight_grad_act8(dy, kept, bias=True)
            assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_offsets_past_32_bits():
    """Gradients and kept rows that lie more than 2^32 bytes from the first, and a dweight of that size."""
    wide = torch.zeros(2 ** 31 // 1024 + 5, 1024 + 8, device="cuda", dtype=torch.bfloat16)  # 4.3 GB
    tokens = wide.shape[0]
    g = torch.Generator(device="cuda").manual_seed(0)
    few = [0, 1, tokens // 2, tokens - 2, tokens - 1]
    x = torch.zeros(tokens, 2080, device="cuda", dtype=torch.bfloat16)  # kept in 4.4 GB
    for t in few:
        wide[t] = torch.randn(1032, device="cuda", generator=g)
        x[t] = torch.randn(2080, device="cuda", generator=g)
    kept = quantize_activation(x)
    small, x = (wide[few][:, 3:43]).contiguous(), x[few].contiguous()
    dw, db = weight_grad_act8(wide[:, 3:43], kept, bias=True)
    check(small, x, dw, db)
    del wide, kept
    torch.cuda.empty_cache()
    dy = torch.zeros(2, 2 ** 31 // 2048 + 300, device="cuda", dtype=torch.bfloat16)
    dy[:, :100], dy[:, -100:] = torch.randn(2, 100, device="cuda", generator=g), torch.randn(2, 100, device="cuda", generator=g)
    x = activations(2, 2048, dtype=torch.bfloat16)
    dw, _ = weight_grad_act8(dy, quantize_activation(x))
    check(dy[:, :100].contiguous(), x, dw[:100])
    check(dy[:, -100:].contiguous(), x, dw[-100:])
    assert not bool(dw[-300:-100].any())


def test_another_stream_and_a_captured_graph():
    dy, x = make(3000, 48, 300, torch.bfloat16)
    kept = quantize_activation(x)
    want = weight_grad_act8(dy, kept, bias=True)
    side = side_stream()
    side.wait_stream(torch.cuda.current_stream())
    got = weight_grad_act8(dy, kept, bias=True, stream=side)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = weight_grad_act8(dy, kept, bias=True)
    for seed in (5, 6, 7):
        dy.copy_(make(3000, 48, 300, torch.bfloat16, seed=seed)[0])
        graph.replay()
        eager = weight_grad_act8(dy, kept, bias=True)
        assert torch.equal(captured[0], eager[0]) and torch.equal(captured[1], eager[1])


def test_refusals():
    dy, x = make(6, 10, 64, torch.bfloat16)
    kept = quantize_activation(x)
    bad = [lambda: weight_grad_act8(dy.float(), kept), lambda: weight_grad_act8(dy[:5], kept), lambda: weight_grad_act8(dy.cpu(), kept),
           lambda: weight_grad_act8(dy, kept, out_dtype=torch.float64), lambda: weight_grad_act8(dy[0, 0], kept),
           lambda: weight_grad_act8(dy.view(2, 3, 10), kept), lambda: weight_grad_act8(dy, kept._replace(features=70))]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    with pytest.raises(RuntimeError, match="no gradient"):
        weight_grad_act8(dy.clone().requires_grad_(), kept)


# ── the layer ────────────────────────────────────────────────────────────────


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("with_bias", [False, True])
def test_linear(dtype, with_bias):
    x = activations(3, 50, 100, dtype=dtype)
    w = (0.1 * activations(40, 100, seed=1)).to(dtype).requires_grad_()
    b = activations(1, 40, dtype=dtype, seed=2)[0].requires_grad_() if with_bias else None
    dy = activations(3, 50, 40, dtype=dtype, seed=3)
    leaf = x.clone().requires_grad_()
    y = linear_act8(leaf, w, b)
    assert torch.equal(y, F.linear(x, w, b))
    inputs = (leaf, w) if b is None else (leaf, w, b)
    got = torch.autograd.grad(y, inputs, dy)
    exact = (dy.double().view(150, 40) @ w.detach().double()).view(3, 50, 100)
    size = (dy.double().abs().view(150, 40) @ w.detach().double().abs()).view(3, 50, 100)
    close(got[0], exact, size, 40, "dx")
    check(dy, x, *got[1:])


@pytest.mark.parametrize("want", ["x", "weight", "bias", "weight bias", "x bias"])
def test_only_some_gradients(want):
    x, w, b = activations(30, 64), activations(20, 64, seed=1), activations(1, 20, seed=2)[0]
    for name, t in (("x", x), ("weight", w), ("bias", b)):
        t.requires_grad_(name in want.split())
    y = linear_act8(x, w, b)
    dy = torch.randn(30, 20, device="cuda")
    y.backward(dy)
    for name, t in (("x", x), ("weight", w), ("bias", b)):
        assert (t.grad is not None) == (name in want.split())
    if w.grad is not None:
        check(dy, x.detach(), w.grad)
    if b.grad is not None:
        close(b.grad, dy.double().sum(0), dy.double().abs().sum(0), 30, "dbias")


def test_layers_share_what_is_kept():
    x = activations(2, 40, 96, dtype=torch.bfloat16)
    kept = quantize_activation(x)
    weights = [(0.1 * activations(24, 96, seed=i)).bfloat16().requires_grad_() for i in range(3)]
    dy = activations(2, 40, 24, dtype=torch.bfloat16, seed=9)
    x.requires_grad_()
    y = sum(linear_act8(x, w, kept=kept) for w in weights)
    grads = torch.autograd.grad(y, weights, dy)
    for g in grads:
        check(dy, x.detach(), g)
    with pytest.raises(ValueError, match="kept is of a"):
        linear_act8(x[:1], weights[0], kept=kept)
    with pytest.raises(ValueError, match="kept is of a"):
        linear_act8(x.float(), weights[0].float(), kept=kept)


def test_a_weight_used_twice_and_autocast():
    x, w = activations(30, 64), (0.1 * activations(64, 64, seed=1)).requires_grad_()
    y = linear_act8(linear_act8(x, w), w)
    h = F.linear(x, w).detach()
    dy = torch.randn(30, 64, device="cuda")
    y.backward(dy)
    dh = dy @ w.detach()
    a, b = products(dy, oracle.kept_values(h)), products(dh, oracle.kept_values(x))
    # dh and h are float32 products of 64 terms each: their own error, 64 * 2^-24, once more
    close(w.grad, a[0] + b[0], a[1] + b[1], 30 + 64 + 64, "dweight")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = linear_act8(x, w)
        assert y.dtype == torch.bfloat16 and torch.equal(y, F.linear(x, w))
    dy = torch.randn(30, 64, device="cuda").bfloat16()
    g, = torch.autograd.grad(y, (w,), dy)
    assert g.dtype == torch.float32
    rounded, _ = weight_grad_act8(dy, quantize_activation(x.bfloat16()))
    assert torch.equal(g, rounded.float())


def test_second_derivatives_and_wrong_arguments_of_the_layer_are_refused():
    x, w = activations(5, 64).requires_grad_(), activations(8, 64, seed=1).requires_grad_()
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(linear_act8(x, w).square().sum(), (x,), create_graph=True)
    for call in (lambda: linear_act8(x, w.bfloat16()), lambda: linear_act8(x, w[:, :63]), lambda: linear_act8(x, w, w[0]),
                 lambda: linear_act8(x.double(), w.double()), lambda: linear_act8(x, w.cpu()), lambda: linear_act8(x, w[0])):
        with pytest.raises(ValueError):
            call()


# ── recomputation ────────────────────────────────────────────────────────────


def block(x, w, u, drop=0.0):
    h = F.gelu(F.linear(x, w))
    if drop:
        h = F.dropout(h, drop)
    return x + F.linear(h, u)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("needs_grad", [True, False])
def test_recomputation_gives_the_gradients_at_the_kept_input(dtype, needs_grad):
    x = activations(2, 30, 64, dtype=dtype).requires_grad_(needs_grad)
    w = (0.1 * activations(96, 64, seed=1)).to(dtype).requires_grad_()
    u = (0.1 * activations(64, 96, seed=2)).to(dtype).requires_grad_()
    dy = activations(2, 30, 64, dtype=dtype, seed=3)
    inputs = (x, w, u) if needs_grad else (w, u)
    y = checkpoint_act8(block, x, w, u)
    assert torch.equal(y, block(x, w, u))
    got = torch.autograd.grad(y, inputs, dy)
    at = quantize_activation(x.detach()).dequantize().requires_grad_(needs_grad)
    want = torch.autograd.grad(block(at, w, u), (at, w, u) if needs_grad else (w, u), dy)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_recomputation_restores_the_random_state_and_keeps_a_byte_a_value():
    x = activations(64, 512, 512, dtype=torch.bfloat16).requires_grad_()
    w = (0.05 * activations(512, 512, seed=1)).bfloat16().requires_grad_()
    u = (0.05 * activations(512, 512, seed=2)).bfloat16().requires_grad_()
    dy = activations(64, 512, 512, dtype=torch.bfloat16, seed=3)
    torch.manual_seed(5)
    y = checkpoint_act8(block, x, w, u, drop=0.5)
    got = torch.autograd.grad(y, (x, w, u), dy)
    del y
    torch.manual_seed(5)
    at = quantize_activation(x.detach()).dequantize().requires_grad_()
    want = torch.autograd.grad(block(at, w, u, drop=0.5), (at, w, u), dy)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    del got, want, at
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    h = checkpoint_act8(block, x * 1, w, u)  # the input itself is not held
    kept = torch.cuda.memory_allocated() - before - h.numel() * 2
    assert kept <= h.numel() * 1.04 + (1 << 20)
    h = checkpoint_act8(block, h, w, u)
    kept = torch.cuda.memory_allocated() - before - h.numel() * 2
    assert kept <= 2 * (h.numel() * 1.04 + (1 << 20))
    h.backward(dy)
    assert x.grad is not None and w.grad is not None


def test_recomputation_without_gradients_and_with_what_it_cannot_keep():
    x, w, u = activations(5, 64), activations(8, 64, seed=1), activations(64, 8, seed=2)
    with torch.no_grad():
        assert torch.equal(checkpoint_act8(block, x.cpu(), w.cpu(), u.cpu()), block(x.cpu(), w.cpu(), u.cpu()))
    with pytest.raises(ValueError):
        checkpoint_act8(block, x.double().requires_grad_(), w, u)
    with pytest.raises(ZeroDivisionError):
        checkpoint_act8(lambda t: t * (1 // 0), x.requires_grad_())
