"""Query/key norms with the position rotation, forward and backward, against formulas in 64 bits and
against differences.

Tolerances, with u = 2^-24 and v the unit roundoff of the type written: a normed value carries the
roundings of the mean of squares (at most log2(dim) + 8 additions), the square root and three products,
which 24 u covers; a rotated one is a sum of two such, |n0| + |n1|. A gradient is r (h - x^ m) with m the mean
of h x^ over the head: 48 u of r (|h| + |x^| mean|h x^|). A weight's gradient is a sum over R rows whose
partial sums round at random: u (64 + 8 sqrt(R)) of the sum of magnitudes. Each plus v of the value and
the type's smallest step.
"""
from __future__ import annotations

import itertools

import pytest
import torch

from stagehand_amd.qk_norm import qk_norm_rope

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -149}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def tables(rows, rot):
    f = 10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64) * 2 / max(rot, 1))
    a = torch.arange(rows, dtype=torch.float64)[:, None] * f
    return a.cos().float().cuda(), a.sin().float().cuda()


def pairs(dim, rot, interleaved):
    p = torch.arange(rot // 2)
    return (2 * p, 2 * p + 1) if interleaved else (p, p + rot // 2)


def angles(cos, sin, positions, start, seq):
    pos = torch.arange(start, start + seq) if positions is None else positions.cpu().long()
    c, s = cos.double().cpu()[pos], sin.double().cpu()[pos]
    return (c, s) if c.dim() == 2 else (c[:, None], s[:, None])


def reference(x, w, cos, sin, positions=None, start=0, interleaved=False, eps=1e-6, dy=None):
    """Float64 results on the CPU: y and its scale, and with dy the gradients and theirs."""
    x = x.detach().double().cpu()
    dim = x.shape[-1]
    w = torch.ones(dim, dtype=torch.float64) if w is None else w.detach().double().cpu()
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    n = x * r * w
    y, size = n.clone(), n.abs()
    rot = 0 if cos is None else 2 * cos.shape[1]
    if rot:
        a, b = pairs(dim, rot, interleaved)
        c, s = angles(cos, sin, positions, start, x.shape[2])
        y[..., a], y[..., b] = n[..., a] * c - n[..., b] * s, n[..., b] * c + n[..., a] * s
        size[..., a] = size[..., b] = n[..., a].abs() + n[..., b].abs()
    if dy is None:
        return y, size
    g = dy.detach().double().cpu().clone()
    gsize = g.abs()
    if rot:
        d = g.clone()
        g[..., a], g[..., b] = d[..., a] * c + d[..., b] * s, d[..., b] * c - d[..., a] * s
        gsize[..., a] = gsize[..., b] = d[..., a].abs() + d[..., b].abs()
    xh, h = x * r, g * w
    dx = r * (h - xh * (h * xh).mean(-1, keepdim=True))
    hs = gsize * w.abs()
    dxs = r * (hs + xh.abs() * (hs * xh.abs()).mean(-1, keepdim=True))
    return y, size, dx, dxs, (g * xh).sum((0, 1, 2)), (gsize * xh.abs()).sum((0, 1, 2))


def close(got, want, slack, what):
    dt = got.dtype
    err = (got.double().cpu() - want).abs()
    bad = ~(err <= slack + ROUND[dt] * want.abs() + TINY[dt])
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(err.max())}"


def check_forward(y, x, w, **kw):
    want, size = reference(x, w, **kw)
    close(y, want, 24 * U * size, "y")


def make(b, hq, hk, s, d, dtype, wdtype=None, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    qkv = (torch.randn(b, s, hq + 2 * hk, d, device="cuda", generator=g) * 2).to(dtype)
    q, k = qkv[:, :, :hq].transpose(1, 2), qkv[:, :, hq:hq + hk].transpose(1, 2)
    wq = (1 + 0.3 * torch.randn(d, device="cuda", generator=g)).to(wdtype or dtype)
    wk = (1 + 0.3 * torch.randn(d, device="cuda", generator=g)).to(wdtype or dtype)
    return q, k, wq, wk


CASES = [  # batch, q heads, k heads, seq, dim, rot
    (1, 1, 1, 1, 2, 2), (1, 2, 1, 3, 4, 2), (2, 3, 3, 5, 6, 6), (1, 4, 2, 33, 16, 16), (3, 2, 2, 7, 24, 8),
    (2, 8, 2, 1, 128, 128), (1, 24, 24, 77, 128, 128), (1, 3, 1, 65, 64, 64), (2, 5, 5, 19, 72, 72), (2, 5, 5, 19, 72, 36),
    (1, 10, 5, 31, 80, 32), (1, 6, 2, 40, 96, 96), (1, 2, 2, 17, 256, 256), (1, 2, 1, 9, 256, 128), (1, 1, 1, 5, 512, 512),
    (1, 2, 2, 6, 510, 200), (1, 3, 3, 4, 130, 34), (4, 1, 7, 12, 32, 32), (1, 2, 2, 10, 128, 0), (1, 2, 2, 10, 20, 0),
    (17, 32, 8, 1, 128, 64),
]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,hq,hk,s,d,rot", CASES)
def test_forward(b, hq, hk, s, d, rot, dtype, interleaved):
    q, k, wq, wk = make(b, hq, hk, s, d, dtype)
    cos, sin = tables(s + 3, rot)
    qo, ko = qk_norm_rope(q, k, wq, wk, cos, sin, start=2, interleaved=interleaved)
    assert qo.is_contiguous() and qo.shape == q.shape and ko.dtype == dtype
    kw = dict(cos=cos if rot else None, sin=sin, start=2, interleaved=interleaved)
    check_forward(qo, q, wq, **kw)
    check_forward(ko, k, wk, **kw)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,hq,hk,s,d,rot", CASES)
def test_backward(b, hq, hk, s, d, rot, dtype, interleaved):
    q, k, wq, wk = (t.requires_grad_() for t in make(b, hq, hk, s, d, dtype, seed=1))
    cos, sin = tables(s, rot)
    qo, ko = qk_norm_rope(q, k, wq, wk, cos, sin, interleaved=interleaved)
    gq, gk = torch.randn_like(qo), torch.randn_like(ko)
    got = torch.autograd.grad((qo, ko), (q, k, wq, wk), (gq, gk))
    for x, w, dy, dx, dw in ((q, wq, gq, got[0], got[2]), (k, wk, gk, got[1], got[3])):
        _, _, want, size, want_w, size_w = reference(x, w, cos if rot else None, sin, interleaved=interleaved, dy=dy)
        close(dx, want, 48 * U * size, "dx")
        rows = x.shape[0] * x.shape[1] * x.shape[2]
        close(dw, want_w, U * (64 + 8 * rows ** 0.5) * size_w, "dweight")


@pytest.mark.parametrize("xdt,wdt", [p for p in itertools.product(DTYPES, DTYPES) if p[0] != p[1]])
def test_weights_of_another_type(xdt, wdt):
    q, k, wq, wk = make(2, 4, 2, 21, 64, xdt, wdt, seed=2)
    cos, sin = tables(21, 64)
    wq.requires_grad_(), wk.requires_grad_()
    qo, ko = qk_norm_rope(q, k, wq, wk, cos, sin)
    check_forward(qo, q, wq, cos=cos, sin=sin)
    gq = torch.randn_like(qo)
    dwq, = torch.autograd.grad((qo * gq).sum(), (wq,))
    assert dwq.dtype == wdt
    _, _, _, _, want, size = reference(q, wq, cos, sin, dy=gq)
    close(dwq, want, U * (64 + 8 * 168 ** 0.5) * size, "dweight")


@pytest.mark.parametrize("pdt", [torch.int32, torch.int64])
@pytest.mark.parametrize("shape", ["seq", "batch", "one", "strided"])
def test_positions(shape, pdt):
    b, s = 3, 11
    q, k, wq, wk = make(b, 4, 2, s, 64, torch.float32, seed=3)
    cos, sin = tables(100, 64)
    p = torch.randint(0, 100, (b, s, 2), device="cuda", dtype=pdt)
    p = {"seq": p[0, :, 0].contiguous(), "batch": p[..., 0].contiguous(), "one": p[:1, :, 0].contiguous(), "strided": p[..., 1]}[shape]
    qo, ko = qk_norm_rope(q, k, wq, wk, cos, sin, positions=p)
    ref = p if p.dim() == 1 or p.shape[0] == b else p[0]
    check_forward(qo, q, wq, cos=cos, sin=sin, positions=ref)
    check_forward(ko, k, wk, cos=cos, sin=sin, positions=ref)


def test_positions_outside_the_tables_give_nan_for_their_tokens():
    q, k, wq, wk = (t.requires_grad_() for t in make(2, 3, 1, 6, 32, torch.float32, seed=4))
    cos, sin = tables(10, 16)
    p = torch.tensor([[0, 9, 10, 3, -1, 2], [1, 2, 3, 2 ** 40, 5, -2 ** 40]], device="cuda")
    qo, ko = qk_norm_rope(q, k, wq, wk, cos, sin, positions=p)
    wrong = (p < 0) | (p >= 10)
    for y, x, w in ((qo, q, wq), (ko, k, wk)):
        rows = wrong[:, None, :].expand(y.shape[:3])
        assert y[rows][:, :16].isnan().all()
        fine = torch.where(wrong, torch.zeros_like(p), p)
        want, size = reference(x, w, cos, sin, positions=fine)
        keep = ~rows.cpu()
        close(y.detach().cpu()[keep], want[keep], 24 * U * size[keep], "y")
    dq, = torch.autograd.grad(qo.sum() + ko.sum(), (q,))
    assert dq[wrong[:, None, :].expand(dq.shape[:3])].isnan().all()
    assert not dq[~wrong[:, None, :].expand(dq.shape[:3])].isnan().any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_zero_infinite_and_nan_heads_stay_their_own(dtype):
    q, k, wq, wk = make(1, 4, 4, 8, 64, dtype, seed=5)
    q = q.clone()
    q[0, 1, 2] = 0
    q[0, 2, 3, 5] = float("inf")
    q[0, 3, 4, 6] = float("nan")
    q[0, 0, 5] = torch.finfo(dtype).tiny
    cos, sin = tables(8, 64)
    qo, _ = qk_norm_rope(q, k, wq, wk, cos, sin)
    assert not qo[0, 1, 2].any()
    assert qo[0, 3, 4].isnan().all()
    bad = torch.zeros(1, 4, 8, dtype=torch.bool)
    bad[0, 2, 3] = bad[0, 3, 4] = True
    want, size = reference(torch.where(bad.cuda()[..., None], torch.ones_like(q), q), wq, cos, sin)
    close(qo.cpu()[~bad], want[~bad], 24 * U * size[~bad], "y")
    assert not torch.isfinite(qo.cpu()[bad]).all(-1).any()


def test_strides_of_inputs_outputs_and_gradients():
    cos, sin = tables(9, 32)
    base = torch.randn(2, 9, 3, 5, 66, device="cuda", dtype=torch.bfloat16)
    w = torch.randn(64, device="cuda", dtype=torch.bfloat16)
    views = [base[:, :, 1, :, 1:65].transpose(1, 2), base[:, :, 0, :, 2:].transpose(1, 2), base[:, :, 2, ::2, :64].permute(0, 2, 1, 3),
             base[:, ::2, 2, :, :64].transpose(1, 2), base[..., :64][:, :, 0].permute(0, 2, 1, 3)[..., ::1],
             base[0, :, 0, :1, :64].transpose(0, 1)[None].expand(3, 4, 9, 64),
             torch.randn(2, 5, 64, 9, device="cuda", dtype=torch.bfloat16).transpose(2, 3)]
    for x in views:
        x = x.detach().requires_grad_()
        y, none = qk_norm_rope(x, None, w, None, cos, sin)
        assert none is None
        check_forward(y, x, w, cos=cos[:x.shape[2]], sin=sin)
        for dy in (torch.randn_like(y), torch.randn(y.shape[0], y.shape[2], y.shape[1], 64, device="cuda").to(y.dtype).transpose(1, 2),
                   torch.ones((), dtype=y.dtype, device="cuda").expand(y.shape)):
            dx, = torch.autograd.grad(y, (x,), dy, retain_graph=True)
            _, _, want, size, _, _ = reference(x, w, cos[:x.shape[2]], sin, dy=dy)
            close(dx, want, 48 * U * size, "dx")


def test_gradients_accumulate_through_a_shared_projection_and_a_shared_weight():
    """q and k as views of one leaf, one weight for both, heads expanded from one: autograd's own sums apply."""
    cos, sin = tables(12, 64)
    qkv = torch.randn(2, 12, 3, 4, 64, device="cuda", requires_grad=True)
    w = (1 + 0.1 * torch.randn(64, device="cuda")).requires_grad_()
    q, k, v = (t.transpose(1, 2) for t in qkv.unbind(2))
    qo, ko = qk_norm_rope(q, k[:, :1].expand(2, 4, 12, 64), w, w, cos, sin, interleaved=True)
    gq, gk = torch.randn_like(qo), torch.randn_like(ko)
    ((qo * gq).sum() + (ko * gk).sum()).backward()
    _, _, dq, sq, dwq, swq = reference(q, w, cos, sin, interleaved=True, dy=gq)
    _, _, dk, sk, dwk, swk = reference(k[:, :1].expand(2, 4, 12, 64), w, cos, sin, interleaved=True, dy=gk)
    close(qkv.grad[:, :, 0].transpose(1, 2), dq, 48 * U * sq, "dq")
    close(qkv.grad[:, :, 1, :1].transpose(1, 2), dk.sum(1, keepdim=True), 64 * U * sk.sum(1, keepdim=True), "dk")
    assert not qkv.grad[:, :, 1, 1:].any() and not qkv.grad[:, :, 2].any()
    close(w.grad, dwq + dwk, U * (66 + 8 * 96 ** 0.5) * (swq + swk), "dweight")


@pytest.mark.parametrize("want", ["q", "k", "qw", "kw", "q kw", "one output"])
def test_only_some_gradients(want):
    q, k, wq, wk = make(2, 3, 2, 7, 64, torch.float32, seed=6)
    cos, sin = tables(7, 64)
    leaf = {"q": q, "k": k, "qw": wq, "kw": wk}
    names = ["q", "k"] if want == "one output" else want.split()
    for n in names:
        leaf[n].requires_grad_()
    qo, ko = qk_norm_rope(q, k, wq, wk, cos, sin)
    gq, gk = torch.randn_like(qo), torch.randn_like(ko)
    loss = (ko * gk).sum() if want == "one output" else (qo * gq).sum() + (ko * gk).sum()
    got = dict(zip(names, torch.autograd.grad(loss, [leaf[n] for n in names], allow_unused=True)))
    if want == "one output":
        gq = torch.zeros_like(gq)
    for n in names:
        x, w, dy = (q, wq, gq) if n[0] == "q" else (k, wk, gk)
        _, _, dx, sx, dw, sw = reference(x, w, cos, sin, dy=dy)
        if len(n) == 1:
            close(got[n], dx, 48 * U * sx, n)
        else:
            close(got[n], dw, U * (64 + 8 * 42 ** 0.5) * sw, n)


def test_gradients_match_differences():
    """Directional differences of a loss in float64 of the float32 outputs. With steps of 2^-6 the cubic term
    is under 1e-3 of the derivative's scale, and the outputs' rounding (2^-24 of ~1000 values, over the step)
    under 1e-4: 3e-3 of the norm of the terms."""
    q, k, wq, wk = make(1, 2, 2, 5, 48, torch.float32, seed=7)
    q, k = q.contiguous(), k.contiguous()
    cos, sin = tables(5, 24)
    leaves = [t.clone().requires_grad_() for t in (q, k, wq, wk)]
    g = [torch.randn_like(q).double(), torch.randn_like(k).double()]

    def loss(args):
        with torch.no_grad():
            qo, ko = qk_norm_rope(*args, cos, sin)
        return float((qo.double() * g[0]).sum() + (ko.double() * g[1]).sum())

    qo, ko = qk_norm_rope(*leaves, cos, sin)
    grads = torch.autograd.grad((qo, ko), leaves, [t.float() for t in g])
    gen = torch.Generator(device="cuda").manual_seed(8)
    for i, grad in enumerate(grads):
        for _ in range(4):
            d = torch.randn(leaves[i].shape, device="cuda", generator=gen)
            step = 2.0 ** -6
            up = [t.detach() + step * d if j == i else t.detach() for j, t in enumerate(leaves)]
            down = [t.detach() - step * d if j == i else t.detach() for j, t in enumerate(leaves)]
            numeric = (loss(up) - loss(down)) / (2 * step)
            terms = grad.double() * d.double()
            assert abs(numeric - float(terms.sum())) <= 3e-3 * float(terms.norm() * terms.numel() ** 0.5 + 1)


def test_out_and_in_place():
    q, k, wq, wk = make(2, 4, 2, 10, 128, torch.bfloat16, seed=9)
    cos, sin = tables(10, 128)
    want = qk_norm_rope(q, k, wq, wk, cos, sin)
    joint_q = torch.full((2, 4, 16, 128), 3.0, device="cuda", dtype=torch.bfloat16)
    joint_k = torch.full((2, 2, 16, 128), 3.0, device="cuda", dtype=torch.bfloat16)
    got = qk_norm_rope(q, k, wq, wk, cos, sin, out=(joint_q[:, :, 4:14], joint_k[:, :, 4:14]))
    for o, w, joint in zip(got, want, (joint_q, joint_k)):
        assert torch.equal(o, w)
        assert bool((joint[:, :, :4] == 3).all()) and bool((joint[:, :, 14:] == 3).all())
    qi, ki = q.clone(), k.clone()
    qk_norm_rope(qi, ki, wq, wk, cos, sin, out=(qi, ki))
    assert torch.equal(qi, want[0]) and torch.equal(ki, want[1])


def test_second_derivatives_are_refused():
    q, k, wq, wk = (t.requires_grad_() for t in make(1, 2, 2, 4, 32, torch.float32))
    qo, ko = qk_norm_rope(q, k, wq, wk)
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(qo.square().sum(), (q,), create_graph=True)


def test_nothing_to_do():
    w = torch.ones(64, device="cuda", requires_grad=True)
    cos, sin = tables(4, 64)
    for shape in ((0, 2, 4, 64), (1, 2, 0, 64), (1, 0, 4, 64)):
        x = torch.empty(shape, device="cuda", requires_grad=True)
        y, _ = qk_norm_rope(x, None, w, None, cos, sin)
        assert y.shape == shape
        dx, dw = torch.autograd.grad(y.sum(), (x, w))
        assert dx.shape == shape and not dw.any()


def test_long_sums_and_repeated_calls():
    """Many rows over many workgroups: the weights' gradients in a fixed order, equal bit for bit."""
    q, k, wq, wk = (t.requires_grad_() for t in make(2, 12, 3, 3001, 64, torch.bfloat16, torch.float32, seed=10))
    cos, sin = tables(3001, 64)
    gq = torch.randn(q.shape, device="cuda").to(q.dtype)
    gk = torch.randn(k.shape, device="cuda").to(k.dtype)
    runs = [torch.autograd.grad(qk_norm_rope(q, k, wq, wk, cos, sin), (q, k, wq, wk), (gq, gk)) for _ in range(3)]
    for x, w, dy, dx, dw in ((q, wq, gq, runs[0][0], runs[0][2]), (k, wk, gk, runs[0][1], runs[0][3])):
        _, _, want, size, want_w, size_w = reference(x, w, cos, sin, dy=dy)
        close(dx, want, 48 * U * size, "dx")
        close(dw, want_w, U * (64 + 8 * (x.numel() / 64) ** 0.5) * size_w, "dweight")
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_offsets_past_32_bits():
    q = torch.zeros(1, 40, 850000, 128, dtype=torch.bfloat16, device="cuda")  # 4.35 G values
    tail = torch.randn(1, 2, 5, 128, device="cuda").to(torch.bfloat16)
    q[:, -2:, -5:] = tail
    w = torch.randn(128, device="cuda").to(torch.bfloat16)
    cos, sin = tables(850000, 128)
    y, _ = qk_norm_rope(q, None, w, None, cos, sin)
    want, size = reference(tail, w, cos[-5:], sin[-5:])
    close(y[:, -2:, -5:], want, 24 * U * size, "y")
    assert not bool(y[:, :38].any()) and not bool(y[:, 38:, :-5].any())


@pytest.mark.parametrize("grad", [False, True])
def test_another_stream_and_a_captured_graph(grad):
    q, k, wq, wk = make(2, 4, 2, 50, 64, torch.bfloat16, seed=11)
    cos, sin = tables(50, 64)
    want = qk_norm_rope(q, k, wq, wk, cos, sin)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = qk_norm_rope(q, k, wq, wk, cos, sin, stream=side)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    fixed = q.clone().requires_grad_(grad)
    wg = wq.clone().requires_grad_(grad)
    gq, gk = torch.randn_like(want[0]), torch.randn_like(want[1])

    def step(x, w):
        qo, ko = qk_norm_rope(x, k, w, wk, cos, sin)
        return (qo, ko, *torch.autograd.grad((qo,), (x, w), (gq,))) if grad else (qo, ko)

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(fixed, wg)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(fixed, wg)
    for n in range(3):
        with torch.no_grad():
            fixed.copy_(q * (n + 1) + n)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, step(fixed, wg)):
            assert torch.equal(a, b)


def test_refusals():
    q, k, wq, wk = make(2, 4, 2, 6, 64, torch.bfloat16)
    cos, sin = tables(8, 64)
    p = torch.zeros(6, dtype=torch.int64, device="cuda")
    bad = [
        lambda: qk_norm_rope(q[0], k, wq, wk, cos, sin), lambda: qk_norm_rope(q.double(), k.double(), wq, wk, cos, sin),
        lambda: qk_norm_rope(q.cpu(), k, wq, wk, cos, sin), lambda: qk_norm_rope(q, k.float(), wq, wk, cos, sin),
        lambda: qk_norm_rope(q, k[:, :, :5], wq, wk, cos, sin), lambda: qk_norm_rope(q, k[:1], wq, wk, cos, sin),
        lambda: qk_norm_rope(q[..., :63], k[..., :63]), lambda: qk_norm_rope(q.repeat(1, 1, 1, 9), None),
        lambda: qk_norm_rope(q, None, wq, wk), lambda: qk_norm_rope(q, k, wq[:32], wk), lambda: qk_norm_rope(q, k, wq, wk.float()),
        lambda: qk_norm_rope(q, k, wq.cpu(), wk), lambda: qk_norm_rope(q, k, wq, wk, cos), lambda: qk_norm_rope(q, k, wq, wk, cos, sin.double()),
        lambda: qk_norm_rope(q, k, wq, wk, cos, sin[:7]), lambda: qk_norm_rope(q, k, wq, wk, *tables(8, 128)),
        lambda: qk_norm_rope(q, k, wq, wk, cos, sin, start=3), lambda: qk_norm_rope(q, k, wq, wk, cos, sin, start=-1),
        lambda: qk_norm_rope(q, k, wq, wk, cos, sin, positions=p[:5]), lambda: qk_norm_rope(q, k, wq, wk, cos, sin, positions=p.float()),
        lambda: qk_norm_rope(q, k, wq, wk, cos, sin, positions=p.cpu()), lambda: qk_norm_rope(q, k, wq, wk, positions=p),
        lambda: qk_norm_rope(q, k, wq, wk, cos, sin, positions=p, start=1), lambda: qk_norm_rope(q, k, wq, wk, cos, sin, eps=-1.0),
        lambda: qk_norm_rope(q, k, wq, wk, cos, sin, eps=float("nan")), lambda: qk_norm_rope(q, k, wq, wk, cos, sin, eps=1e40),
        lambda: qk_norm_rope(q, k, wq, wk, cos.clone().requires_grad_(), sin),
        lambda: qk_norm_rope(q, k, wq, wk, cos, sin, out=(torch.empty_like(q), None)),
        lambda: qk_norm_rope(q, k, wq, wk, cos, sin, out=(torch.empty_like(q).float(), torch.empty_like(k))),
        lambda: qk_norm_rope(q, k, wq, wk, cos, sin, out=(torch.empty(2, 4, 64, 6, device="cuda", dtype=q.dtype).transpose(2, 3), torch.empty_like(k))),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    with pytest.raises(RuntimeError, match="no gradient"):
        qk_norm_rope(q.clone().requires_grad_(), k, wq, wk, cos, sin, out=(torch.empty_like(q), torch.empty_like(k)))
