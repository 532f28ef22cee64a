"""Layer norms, forward and backward, against formulas in 64 bits and against differences.

Tolerances, with u = 2^-24 and M = mean |x|: a row's sum takes at most 16 additions in a work-item, 6 in a wavefront and
16 over wavefronts, so a mean is off by 40 u M (with its division), a variance by 45 u of itself and the
square of the mean's error, e = 40 u M r in units of the norm: n is off by E = |n| (36 u + e^2) + 44 u M r. With g = dy w: y by |w| E + 4 u (|n w| +
|b|); dx = r (g - mean g - n mean(g n)) by r (48 u (|g| + mean |g| + |n| mean |g n|) + |n| mean(|g| E) + E mean |g n|) and the error
36 u + e^2 of r itself; a sum over R tokens, whose partial sums round at random, by u (64 + 8 sqrt(R)) of the sum of magnitudes,
dweight's also by sum |dy| E. Each plus half a step of the type written.
"""
from __future__ import annotations

import act8_oracle as oracle
import pytest
import torch
from act8_oracle import DTYPES, ROUND, TINY, activations
from side_stream import side_stream

from stagehand_amd.act8 import quantize_activation
from stagehand_amd.layer_norm import layer_norm

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = 1e-6
CASES = [  # batch, seq, features: every shape of rows, with and without ragged ends
    (1, 1, 1), (1, 3, 2), (2, 5, 7), (1, 1, 64), (3, 17, 40), (1, 9, 512), (2, 6, 513), (1, 33, 1000), (2, 3, 1024), (1, 5, 1155),
    (1, 2, 2048), (3, 7, 2056), (2, 9, 4096), (1, 4, 4097), (1, 6, 8192), (1, 3, 8200), (2, 2, 16384), (1, 3, 16383), (70, 1, 96), (2, 2100, 128),
    (1, 1300, 1536), (5, 300, 600),
]


def close(got, want, slack, what):
    err = (got.double() - want).abs()
    bad = ~(err <= slack + ROUND[got.dtype] * want.abs() + TINY[got.dtype])
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(err.max())}"


def reference(x, w, b, dy=None, modulate=False, eps=EPS, kept=None):
    """(value, slack) of y and, with dy, of dx, dweight and dbias, in 64 bits."""
    x = x.detach().double()
    batch = x.shape[0]
    rows = any(t is not None and t.numel() != x.shape[-1] for t in (w, b))

    def param(t, default):
        if t is None:
            return torch.full((1, 1, x.shape[-1]), default, dtype=torch.float64, device=x.device)
        return t.detach().double().reshape(batch if rows else 1, 1, x.shape[-1])

    wt, bt = param(w, 0.0 if modulate else 1.0), param(b, 0.0)
    if modulate:
        wt = wt + 1
    mean = x.mean(-1, keepdim=True)
    r = 1 / ((x - mean).square().mean(-1, keepdim=True) + eps).sqrt()
    size = x.abs().mean(-1, keepdim=True)
    e = 40 * U * size * r

    def norm(v):
        n = (v - mean) * r
        return n, n.abs() * (36 * U + e * e) + 44 * U * size * r

    n, off = norm(x)
    y = n * wt + bt, wt.abs() * off + 4 * U * ((n * wt).abs() + bt.abs())
    if dy is None:
        return y
    if kept is not None:
        n, off = norm(kept)
    dy = dy.detach().double()
    g = dy * wt
    gn = (g * n).abs().mean(-1, keepdim=True)
    dx = r * (g - g.mean(-1, keepdim=True) - n * (g * n).mean(-1, keepdim=True))
    parts = g.abs() + g.abs().mean(-1, keepdim=True) + n.abs() * gn
    dx_slack = r * (48 * U * parts + n.abs() * (g.abs() * off).mean(-1, keepdim=True) + off * gn) + r * parts * (36 * U + e * e)
    dims = (1,) if rows else (0, 1)
    count = x.shape[1] * (1 if rows else batch)
    share = U * (64 + 8 * count ** 0.5)
    dw = (dy * n).sum(dims), (dy.abs() * off).sum(dims) + share * (dy * n).abs().sum(dims)
    db = dy.sum(dims), share * dy.abs().sum(dims)
    return y, (dx, dx_slack), dw, db


def make(b, s, n, dtype, modulate=False, wdtype=None, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    x = activations(b, s, n, dtype=dtype, seed=seed)
    dy = torch.randn(b, s, n, device="cuda", generator=g).to(dtype)
    if modulate:
        six = (0.3 * torch.randn(b, 1, 6 * n, device="cuda", generator=g)).to(wdtype or dtype).chunk(6, -1)
        return x, six[1], six[0], dy
    w = (1 + 0.1 * torch.randn(n, device="cuda", generator=g)).to(wdtype or dtype)
    return x, w, (0.1 * torch.randn(n, device="cuda", generator=g)).to(wdtype or dtype), dy


def leaves(*tensors):
    return [None if t is None else t.detach().requires_grad_() for t in tensors]


def check(x, w, b, dy, **kw):
    """Forward and backward of leaves that share the memory of x, w and b."""
    xl, wl, bl = leaves(x, w, b)
    y = layer_norm(xl, wl, bl, **kw)
    keep8 = kw.pop("keep8", False)
    kept = oracle.kept_values(x.reshape(-1, x.shape[-1])).view(x.shape).cuda() if keep8 else None
    three = [t.reshape(1, -1, x.shape[-1]) if t is not None and t.dim() != 3 else t for t in (x, dy, kept)]
    want = reference(three[0], w, b, three[1], kept=three[2], **kw)
    with torch.no_grad():
        assert torch.equal(y, layer_norm(x, w, b, **kw))
    inputs = [t for t in (xl, wl, bl) if t is not None]
    got = dict(zip([n for n, t in (("dx", xl), ("dweight", wl), ("dbias", bl)) if t is not None], torch.autograd.grad(y, inputs, dy)))
    close(y.detach(), want[0][0].view(x.shape), want[0][1].view(x.shape), "y")
    close(got["dx"], want[1][0].view(x.shape), want[1][1].view(x.shape), "dx")
    assert got["dx"].shape == x.shape and got["dx"].dtype == x.dtype
    for name, t, i in (("dweight", w, 2), ("dbias", b, 3)):
        if t is not None:
            assert got[name].shape == t.shape and got[name].dtype == t.dtype
            close(got[name], want[i][0].view(t.shape), want[i][1].view(t.shape), name)


@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("modulate", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,s,n", CASES)
def test_forward_and_backward(b, s, n, dtype, modulate, keep8):
    x, w, bias, dy = make(b, s, n, dtype, modulate, seed=n)
    check(x, w, bias, dy, modulate=modulate, keep8=keep8)


@pytest.mark.parametrize("xdt", DTYPES)
@pytest.mark.parametrize("wdt", DTYPES)
def test_weights_of_another_type(xdt, wdt):
    for b, s, n, modulate in ((2, 40, 100, True), (1, 700, 300, False), (2, 3, 4100, False)):
        x, w, bias, dy = make(b, s, n, xdt, modulate, wdt)
        check(x, w, bias, dy, modulate=modulate)


@pytest.mark.parametrize("modulate", [False, True])
@pytest.mark.parametrize("which", ["", "weight", "bias"])
def test_without_weight_or_bias(which, modulate):
    for n in (70, 3000):
        x, w, bias, dy = make(2, 9, n, torch.bfloat16)
        check(x, w if which == "weight" else None, bias if which == "bias" else None, dy, modulate=modulate)
        x, w, bias, dy = make(2, 9, n, torch.float32, True)
        check(x, w if which == "weight" else None, bias if which == "bias" else None, dy, modulate=modulate)


@pytest.mark.parametrize("dtype", DTYPES)
def test_shapes_of_inputs_and_weights(dtype):
    x, w, bias, dy = make(4, 6, 200, dtype)
    for cut in (lambda t: t[0, 0], lambda t: t[0], lambda t: t.view(2, 2, 6, 200), lambda t: t[:, 2], lambda t: t[:, ::2], lambda t: t.transpose(0, 1)):
        check(cut(x), w, bias, cut(dy))
    check(x, w[None], bias[None, None], dy)
    for cut in (slice(3, 68), slice(8, 104), slice(0, 199)):  # columns of wider rows
        check(x[..., cut], w[cut], bias[cut], dy[..., cut])
    check(x[..., ::2], w[::2], bias[::2], dy[..., ::2])
    check(x, w[:1].expand(200), bias[:1].expand(200), dy)
    check(x[:1].expand(4, 6, 200), w, bias, dy[:, :1].expand(4, 6, 200))
    x, w, bias, dy = make(4, 6, 200, dtype, True)
    check(x, w[:, 0], bias[:, 0], dy, modulate=True)
    check(x.transpose(0, 1).contiguous().transpose(0, 1), w.contiguous(), bias, dy, modulate=True)
    check(x[:, :, 3:70], w[..., 3:70], bias[..., 3:70], dy[..., 3:70], modulate=True, keep8=True)


def test_rows_far_from_zero_constant_rows_and_eps():
    x, w, bias, dy = make(1, 20, 700, torch.float32)
    x[0, :5] += 1e4
    x[0, 5] = 3.0
    x[0, 6] = 0.0
    x[0, 7] = 1e-20
    check(x, w, bias, dy)
    check(x, w, bias, dy, eps=1.0)
    y = layer_norm(x, w, bias)
    assert torch.equal(y[0, 6], bias)
    check(x[:, 8:], w, bias, dy[:, 8:], eps=0.0)
    # one feature: a norm of zero
    assert torch.equal(layer_norm(x[..., :1], None, bias[:1]), bias[:1].expand(1, 20, 1))


@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("n", [100, 3000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_broken_tokens_stay_their_own(dtype, n, keep8):
    x, w, bias, dy = make(1, 12, n, dtype)
    x[0, 3, 5], x[0, 7, n - 1], dy[0, 9, 50] = float("nan"), float("inf"), float("nan")
    xl, wl, bl = leaves(x, w, bias)
    y = layer_norm(xl, wl, bl, keep8=keep8)
    dx, dw, db = torch.autograd.grad(y, (xl, wl, bl), dy)
    good = [i for i in range(12) if i not in (3, 7, 9)]
    assert bool(y[0, 3].isnan().all()) and bool(y[0, 7].isnan().all()) and bool(dx[0, 9].isnan().all())
    assert bool(dx[0, 3].isnan().all()) and bool(dx[0, 7].isnan().all())
    xl, = leaves(x[:, good])
    clean = layer_norm(xl, w, bias, keep8=keep8)
    assert torch.equal(y[:, good], clean) and bool(y[0, 9].isfinite().all())
    assert torch.equal(dx[:, good], torch.autograd.grad(clean, (xl,), dy[:, good])[0])
    assert bool(db[:50].isfinite().all()) and bool(db[50].isnan()) and bool(dw.isnan().all())


@pytest.mark.parametrize("want", ["x", "weight", "bias", "x weight", "weight bias"])
@pytest.mark.parametrize("keep8", [False, True])
def test_only_some_gradients(want, keep8):
    x, w, bias, dy = make(2, 300, 200, torch.bfloat16)
    kept = oracle.kept_values(x.view(600, 200)).view(x.shape).cuda() if keep8 else None
    ref = dict(zip(("y", "x", "weight", "bias"), reference(x, w, bias, dy, kept=kept)))
    tensors = {"x": x.clone(), "weight": w.clone(), "bias": bias.clone()}
    for name, t in tensors.items():
        t.requires_grad_(name in want.split())
    layer_norm(tensors["x"], tensors["weight"], tensors["bias"], keep8=keep8).backward(dy)
    for name, t in tensors.items():
        assert (t.grad is not None) == (name in want.split())
        if t.grad is not None:
            close(t.grad, ref[name][0].view(t.shape), ref[name][1].view(t.shape), name)


def test_gradients_match_differences():
    """The forward in fp32, seen through a random linear function in 64 bits, along random directions. With step h the
    difference's own error is h^2 times a third derivative of the order of the gradient, and rounding u / h."""
    for b, s, n, modulate in ((2, 5, 40, False), (2, 5, 1100, True)):
        x, w, bias, _ = make(b, s, n, torch.float32, modulate)
        g = torch.Generator(device="cuda").manual_seed(7)
        c = torch.randn(b, s, n, device="cuda", generator=g)
        xl, wl, bl = leaves(x, w, bias)
        grads = torch.autograd.grad(layer_norm(xl, wl, bl, modulate=modulate), (xl, wl, bl), c)

        def value(p):
            return float((layer_norm(*p, modulate=modulate).double() * c.double()).sum())

        h = 2.0 ** -7
        for i in range(3):
            d = torch.randn(xl.shape if i == 0 else wl.shape, device="cuda", generator=g) if i else \
                torch.randn(xl.shape, device="cuda", generator=g) * x.std()
            up, down = [x, w.contiguous(), bias.contiguous()], [x, w.contiguous(), bias.contiguous()]
            up[i], down[i] = up[i] + h * d, down[i] - h * d
            slope = (value(up) - value(down)) / (2 * h)
            want = float((grads[i].double() * d.double()).sum())
            size = float((grads[i].double() * d.double()).square().sum().sqrt())
            assert abs(slope - want) <= (8 * h * h + 64 * U / h) * max(size, 1.0) * (b * s) ** 0.5, (i, slope, want, size)


def test_out_and_in_place():
    x, w, bias, _ = make(3, 9, 300, torch.bfloat16)
    want = layer_norm(x, w, bias)
    joint = torch.full((3, 20, 320), 7.0, device="cuda", dtype=torch.bfloat16)
    out, version = joint[:, 5:14, 10:310], joint._version
    assert layer_norm(x, w, bias, out=out) is out and torch.equal(out, want) and joint._version > version
    joint[:, 5:14, 10:310] = 7.0
    assert bool((joint == 7).all())
    same = x.clone()
    layer_norm(same, w, bias, out=same)
    assert torch.equal(same, want)
    a = torch.ones(3, 9, 300, device="cuda", requires_grad=True)
    held = torch.ones(3, 9, 300, device="cuda")
    y = a * held
    layer_norm(held.clone(), out=held)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with torch.inference_mode():
        layer_norm(x, out=torch.empty_like(x))


def test_second_derivatives_are_refused():
    x = activations(2, 3, 40).requires_grad_()
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(layer_norm(x).square().sum(), (x,), create_graph=True)


def test_nothing_to_do():
    w, bias = torch.ones(40, device="cuda", requires_grad=True), torch.ones(40, device="cuda", requires_grad=True)
    for shape in ((0, 40), (2, 0, 40), (0, 3, 40)):
        x = torch.empty(shape, device="cuda", requires_grad=True)
        for keep8 in (False, True):
            y = layer_norm(x, w, bias, keep8=keep8)
            assert y.shape == shape
            grads = torch.autograd.grad(y, (x, w, bias), torch.empty(shape, device="cuda"))
            assert grads[0].shape == shape and not grads[1].any() and not grads[2].any()
    x = torch.empty(3, 0, 40, device="cuda", requires_grad=True)
    m = torch.ones(3, 1, 40, device="cuda", requires_grad=True)
    g, = torch.autograd.grad(layer_norm(x, m, modulate=True), (m,), torch.empty(3, 0, 40, device="cuda"))
    assert g.shape == m.shape and not g.any()


def test_what_is_kept_is_a_byte_a_value():
    x, w, bias, dy = make(2, 1000, 4096, torch.bfloat16)
    x.requires_grad_()
    torch.cuda.synchronize()
    used = []
    for keep8 in (False, True):
        before = torch.cuda.memory_allocated()
        y = layer_norm(x * 1, w, bias, keep8=keep8)  # of a tensor that only the norm could hold
        used.append(torch.cuda.memory_allocated() - before - 2 * x.numel())
        del y
    assert used[0] >= 2 * x.numel() and used[1] <= 1.04 * x.numel() + (1 << 20)


def test_repeated_calls_give_the_same_bits():
    for b, s, n, modulate in ((1, 5000, 200, False), (2, 900, 4096, True), (3, 77, 1155, False)):
        x, w, bias, dy = make(b, s, n, torch.bfloat16, modulate)
        xl, wl, bl = leaves(x, w, bias)
        first = torch.autograd.grad(layer_norm(xl, wl, bl, modulate=modulate), (xl, wl, bl), dy)
        for _ in range(3):
            again = torch.autograd.grad(layer_norm(xl, wl, bl, modulate=modulate), (xl, wl, bl), dy)
            assert all(torch.equal(p, q) for p, q in zip(first, again))


@pytest.mark.parametrize("keep8", [False, True])
def test_offsets_past_32_bits(keep8):
    n = 4100
    tokens = 2 ** 32 // n + 9
    x = torch.zeros(tokens, n, dtype=torch.bfloat16, device="cuda")
    some = activations(6, n, dtype=torch.bfloat16)
    x[:2], x[-4:] = some[:2], some[2:]
    w = torch.ones(n, device="cuda", requires_grad=True)
    x.requires_grad_()
    y = layer_norm(x, w, keep8=keep8)
    (want, slack) = reference(some[None], w, None)
    close(torch.cat((y[:2], y[-4:])).detach(), want[0], slack[0], "y")
    assert not bool(y[-5].any())
    dy = torch.zeros_like(y)
    few = torch.randn(6, n, device="cuda", dtype=torch.bfloat16)
    dy[:2], dy[-4:] = few[:2], few[2:]
    del y
    y = layer_norm(x, w, keep8=keep8)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    kept = oracle.kept_values(some)[None].cuda() if keep8 else None
    _, (dx_want, dx_slack), (dw_want, dw_slack), _ = reference(some[None], w, None, few[None], kept=kept)
    close(torch.cat((dx[:2], dx[-4:])), dx_want[0], dx_slack[0], "dx")
    close(dw, dw_want, dw_slack, "dweight")


@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("n", [96, 4096])
def test_another_stream_and_a_captured_graph(n, keep8):
    x, w, bias, dy = make(2, 600, n, torch.bfloat16, True)
    want = layer_norm(x, w, bias, modulate=True)
    side = side_stream()
    side.wait_stream(torch.cuda.current_stream())
    got = layer_norm(x, w, bias, modulate=True, stream=side)
    side.synchronize()
    assert torch.equal(got, want)
    fixed, wl, bl = x.clone().requires_grad_(), w.clone().requires_grad_(), bias.clone().requires_grad_()

    def step():
        y = layer_norm(fixed, wl, bl, modulate=True, keep8=keep8)
        return (y, *torch.autograd.grad(y, (fixed, wl, bl), dy))

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for k in range(3):
        with torch.no_grad():
            fixed.copy_(x * (k + 1) + k)
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(outs, step()):
            assert torch.equal(p, q)


def test_refusals():
    x, w, bias, _ = make(3, 5, 64, torch.bfloat16)
    m = torch.zeros(3, 1, 64, device="cuda", dtype=torch.bfloat16)
    bad = [
        lambda: layer_norm(x.double()), lambda: layer_norm(x.cpu()), lambda: layer_norm(torch.tensor(1.0, device="cuda")),
        lambda: layer_norm(x[..., :0]), lambda: layer_norm(torch.empty(1, 16385, device="cuda")), lambda: layer_norm(x, w[:63]),
        lambda: layer_norm(x, w.cpu()), lambda: layer_norm(x, w.double()), lambda: layer_norm(x, w, bias.float()), lambda: layer_norm(x, m, bias),
        lambda: layer_norm(x, w, m), lambda: layer_norm(x[0], m), lambda: layer_norm(x, m[:2]), lambda: layer_norm(x, m.view(3, 64, 1)),
        lambda: layer_norm(x, m.expand(3, 5, 64)), lambda: layer_norm(x, eps=-1.0), lambda: layer_norm(x, eps=float("nan")),
        lambda: layer_norm(x, eps=1e40), lambda: layer_norm(x, out=torch.empty(3, 5, 63, device="cuda", dtype=x.dtype)),
        lambda: layer_norm(x, out=torch.empty_like(x).float()), lambda: layer_norm(x, out=torch.empty(3, 64, 5, device="cuda", dtype=x.dtype).transpose(1, 2)),
        lambda: layer_norm(x, out=torch.empty(1, 5, 64, device="cuda", dtype=x.dtype).expand(3, 5, 64)),
        lambda: layer_norm(x[0], out=torch.empty(5, 128, device="cuda", dtype=x.dtype)[:, ::2]),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    with pytest.raises(RuntimeError, match="no gradient"):
        layer_norm(x.clone().requires_grad_(), out=torch.empty_like(x))
    with pytest.raises(RuntimeError, match="no gradient"):
        layer_norm(x, out=torch.empty_like(x).requires_grad_())
