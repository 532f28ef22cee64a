"""Activations kept in 8 bits and read back: bit-exact against the format in 64 bits."""
from __future__ import annotations

import act8_oracle as oracle
import pytest
import torch
from act8_oracle import DTYPES, activations
from side_stream import side_stream

from stagehand_amd.act8 import Activation8, quantize_activation

pytestmark = pytest.mark.gpu

SIZES = [(1, 1), (3, 7), (1, 8), (2, 31), (5, 32), (4, 33), (77, 64), (3, 1155), (513, 96), (8, 4096), (1, 16385), (300, 40)]


def same(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Equal values, NaNs at the same places."""
    a, b = a.cpu().double(), b.cpu().double()
    return a.shape == b.shape and bool(((a == b) | (a.isnan() & b.isnan())).all())


def check(x: torch.Tensor, kept: Activation8) -> None:
    rows = x.reshape(-1, x.shape[-1])
    q, e = oracle.quantize(rows)
    assert kept.features == x.shape[-1] and kept.shape == x.shape[:-1] and kept.dtype == x.dtype
    assert torch.equal(kept.exponent.cpu(), e)
    assert torch.equal(kept.q.cpu(), q)
    assert same(kept.dequantize(), oracle.dequantize(q, e, x.shape[-1]).view(x.shape))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,cols", SIZES)
def test_bit_exact(tokens, cols, dtype):
    x = activations(tokens, cols, dtype=dtype, seed=tokens + cols)
    kept = quantize_activation(x)
    check(x, kept)
    assert kept.nbytes == tokens * -(-cols // 32) * 33
    # off by at most half a step
    step = torch.exp2(kept.exponent.double().cpu() - 127).repeat_interleave(32, 1)[:, :cols]
    assert bool(((kept.dequantize().double().cpu() - x.double().cpu()).abs() <= step / 2).all())


def groups_at_the_borders(dtype: torch.dtype) -> torch.Tensor:
    """One group a row: maxima at and next to 127 * 2^k, ties, the ends of the type's range, subnormal and broken values."""
    info, rows = torch.finfo(dtype), []
    step = info.eps
    for k in (-20, -6, -1, 0, 3, 8):
        for top in (127 * 2.0 ** k, 127 * 2.0 ** k * (1 + step), 127 * 2.0 ** k * (1 - step / 2), 128 * 2.0 ** k, 64 * 2.0 ** k):
            row = torch.arange(32, dtype=torch.float64) * 2.0 ** k / 2 - 8 * 2.0 ** k  # halves: ties to even
            row[5] = -top
            rows.append(row)
    for top in (info.max, info.max * (1 - 8 * step), info.max / 2, info.tiny, info.tiny * 3, oracle.TINY[dtype], 7 * oracle.TINY[dtype], 0.0):
        row = torch.linspace(-1, 1, 32, dtype=torch.float64) * top
        row[7] = top
        rows.append(row)
    for bad in (float("inf"), -float("inf"), float("nan")):
        row = torch.linspace(-1, 1, 32, dtype=torch.float64)
        row[9] = bad
        rows.append(row)
    return torch.stack(rows).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_borders_of_the_format(dtype):
    x = groups_at_the_borders(dtype).cuda()
    kept = quantize_activation(x)
    check(x, kept)
    finite = x.isfinite().all(1)
    assert bool(kept.dequantize()[finite].isfinite().all()) and bool(kept.dequantize()[~finite].isnan().all())
    # many groups in a row: each its own
    wide = x.reshape(1, -1)
    check(wide, quantize_activation(wide))


@pytest.mark.parametrize("src", DTYPES)
@pytest.mark.parametrize("dst", DTYPES)
def test_reading_in_another_type_rounds_once(src, dst):
    x = activations(9, 70, dtype=src)
    kept = quantize_activation(x)
    assert torch.equal(kept.dequantize(dst).cpu(), oracle.kept_values(x).to(dst))
    assert kept.dequantize(dst).dtype == dst


def test_views_leading_dims_and_out():
    base = activations(4, 6, 200, dtype=torch.bfloat16)
    for x in (base[:, 1::2, 3:68], base[..., 5:101], base[:, 2], base.transpose(0, 1), base[0, 0], base[:, :, ::3], base[1:1]):
        kept = quantize_activation(x)
        assert same(kept.dequantize(), oracle.kept_values(x.reshape(-1, x.shape[-1])).view(x.shape))
    x = base[:, :, 3:68]
    wide = torch.full((4, 6, 90), 7.0, device="cuda", dtype=torch.bfloat16)
    out, kept = wide[..., 11:76], quantize_activation(x)
    version = wide._version
    assert kept.dequantize(out=out) is out and wide._version > version
    assert same(out, oracle.kept_values(x.reshape(24, 65)).view(4, 6, 65))
    assert bool((wide[..., :11] == 7).all()) and bool((wide[..., 76:] == 7).all())
    assert torch.equal(kept.dequantize(out=torch.empty(4, 6, 65, device="cuda")).cpu(), oracle.kept_values(x.reshape(24, 65)).float().view(4, 6, 65))


def test_nothing_to_do():
    for shape in ((0, 5), (3, 0, 64)):
        kept = quantize_activation(torch.empty(shape, device="cuda"))
        assert kept.dequantize().shape == shape


def test_offsets_past_32_bits():
    cols = 4112
    tokens = 2 ** 32 // cols + 9
    x = torch.zeros(tokens, cols, dtype=torch.bfloat16, device="cuda")
    some = activations(5, cols, dtype=torch.bfloat16)
    x[:2], x[-3:] = some[:2], some[2:]
    kept = quantize_activation(x)
    del x
    want = oracle.kept_values(some)
    y = kept.dequantize()
    assert same(y[:2], want[:2]) and same(y[-3:], want[2:]) and not bool(y[-4].any())


def test_another_stream_and_a_captured_graph():
    x = activations(300, 1155, dtype=torch.bfloat16)
    want = oracle.kept_values(x)
    side = side_stream()
    side.wait_stream(torch.cuda.current_stream())
    kept = quantize_activation(x, stream=side)
    y = kept.dequantize(stream=side.cuda_stream)
    side.synchronize()
    assert same(y, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = quantize_activation(x)
        y = kept.dequantize()
    for seed in (1, 2, 3):
        x.copy_(activations(300, 1155, dtype=torch.bfloat16, seed=seed))
        graph.replay()
        assert same(y, oracle.kept_values(x))
        assert torch.equal(quantize_activation(x).q, kept.q)


def test_refusals():
    x = activations(4, 64)
    kept = quantize_activation(x)
    bad = [lambda: quantize_activation(x.double()), lambda: quantize_activation(x.cpu()), lambda: quantize_activation(x[:, :0]),
           lambda: quantize_activation(torch.tensor(1.0, device="cuda")), lambda: kept.dequantize(torch.float64),
           lambda: kept.dequantize(out=torch.empty(4, 63, device="cuda")), lambda: kept.dequantize(torch.bfloat16, torch.empty(4, 64, device="cuda")),
           lambda: kept.dequantize(out=torch.empty(64, 4, device="cuda").t()),
           lambda: kept._replace(features=65).dequantize(), lambda: kept._replace(features=0).dequantize(),
           lambda: kept._replace(q=kept.q[:3]).dequantize(), lambda: kept._replace(q=kept.q.float()).dequantize(),
           lambda: kept._replace(exponent=kept.exponent.cpu()).dequantize(), lambda: kept._replace(exponent=kept.exponent[:, :1]).dequantize(),
           lambda: kept._replace(q=kept.q.t().contiguous().t()).dequantize(), lambda: kept._replace(dtype=torch.int8).dequantize()]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    with pytest.raises(RuntimeError, match="no gradient"):
        quantize_activation(x.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="no gradient"):
        kept.dequantize(out=torch.empty(4, 64, device="cuda", requires_grad=True))
