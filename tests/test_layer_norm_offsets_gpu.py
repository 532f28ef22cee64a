"""Layer norms of rows whose mean is far above their spread.

The mean of the differences corrects the mean that they are taken from. With u = 2^-24, M = mean |x| and e = 40 u M r (the first mean's error
in units of the norm): a difference rounds by u of itself, and the sums of differences and of their squares take at most 40 additions each,
so n is off by |n| (48 u + 96 u e^2) + 48 u (1 + e), and the variance by 96 u e^2 / r^2 besides its own 48 u. Nothing of it is u M r. The
backward pass takes its mean from memory, as an fp32 number: there n is off by 2 u M r more.
"""
from __future__ import annotations

import pytest
import torch
from act8_oracle import DTYPES
from test_layer_norm_gpu import EPS, U, close

from stagehand_amd.layer_norm import layer_norm

pytestmark = pytest.mark.gpu

COLS = [7, 96, 600, 1155, 2880, 7666, 16383]  # every shape of rows


def params(n, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return 1 + 0.1 * torch.randn(n, device="cuda", generator=g), 0.1 * torch.randn(n, device="cuda", generator=g)


def check(x, w, b, dy):
    xl, wl, bl = (t.clone().requires_grad_() for t in (x, w, b))
    y = layer_norm(xl, wl, bl)
    dx, dw, db = torch.autograd.grad(y, (xl, wl, bl), dy)
    v, dyd, wd, bd = x.double(), dy.double(), w.double(), b.double()
    mean = v.mean(-1, keepdim=True)
    r = 1 / ((v - mean).square().mean(-1, keepdim=True) + EPS).sqrt()
    n, e = (v - mean) * r, 40 * U * v.abs().mean(-1, keepdim=True) * r
    r_off = 48 * U + 96 * U * e * e
    off = n.abs() * r_off + 48 * U * (1 + e)
    close(y.detach(), n * wd + bd, wd.abs() * off + 4 * U * ((n * wd).abs() + bd.abs()), "y")
    assert torch.equal(layer_norm(x, w, b), y.detach())
    off = off + e / 20
    g = dyd * wd
    gn = (g * n).abs().mean(-1, keepdim=True)
    parts = g.abs() + g.abs().mean(-1, keepdim=True) + n.abs() * gn + off * (g.abs() * off).mean(-1, keepdim=True)
    slack = r * (48 * U * parts + n.abs() * (g.abs() * off).mean(-1, keepdim=True) + off * gn + parts * r_off + off * (g.abs() * off).mean(-1, keepdim=True))
    close(dx, r * (g - g.mean(-1, keepdim=True) - n * (g * n).mean(-1, keepdim=True)), slack, "dx")
    share = U * (64 + 8 * x.shape[0] ** 0.5)
    close(dw, (dyd * n).sum(0), (dyd.abs() * off).sum(0) + share * (dyd * n).abs().sum(0), "dweight")
    close(db, dyd.sum(0), share * dyd.abs().sum(0), "dbias")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", COLS)
def test_constant_rows(n, dtype):
    """Their norm is 0, so the output is the bias. The differences are equal, and so small that even r is not off: e <= 40 u 2688 / sqrt(eps)."""
    levels = torch.tensor([100.0, 1000.0, 2688.0, -1776.0, 3.0, -0.2, 0.0], device="cuda").to(dtype)
    x = levels[:, None].expand(-1, n).contiguous()
    w, b = params(n, n)
    off = (48 * U * 40 * U * levels.double().abs() / EPS ** 0.5)[:, None]
    for keep8 in (False, True):
        y = layer_norm(x.clone().requires_grad_(), w, b, keep8=keep8).detach()
        close(y, b.double().expand(x.shape), w.double() * off + 2 * U * b.double().abs(), "y")
        assert torch.equal(layer_norm(x, w, b), y)
    dy = torch.randn(x.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(n)).to(dtype)
    xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(layer_norm(xl, wl, b), (xl, wl), dy)
    g = dy.double() * w.double()
    r, mean = EPS ** -0.5, g.mean(-1, keepdim=True)
    e = 40 * U * levels.double().abs()[:, None] * r
    size = g.abs() + g.abs().mean(-1, keepdim=True)
    # the mean that is kept is the level itself, and n is 0
    close(dx, r * (g - mean), r * size * (48 * U + 96 * U * e * e), "dx")
    assert not dw.any()


@pytest.mark.parametrize("n", COLS)
@pytest.mark.parametrize("level,spread", [(1e4, 1.0), (-3e3, 0.05), (1e6, 40.0), (50.0, 1e-3)])
def test_rows_far_from_zero(n, level, spread):
    g = torch.Generator(device="cuda").manual_seed(n)
    x = level + spread * torch.randn(40, n, device="cuda", generator=g)
    check(x, *params(n, n), torch.randn(40, n, device="cuda", generator=g))
    x = (level + 8 * abs(level) * 2.0 ** -8 * torch.randn(40, n, device="cuda", generator=g)).bfloat16()
    check(x, *params(n, n), torch.randn(40, n, device="cuda", generator=g).bfloat16())
