"""Int8 linear layers against a plain implementation in 64 bits.

Quantised tokens are compared bit for bit with numpy's float32. A product's tolerance is the sum of what
its roundings may be off: with A = |acc| + |zero point * sum| before scaling, u = 2^-24 and v the unit
roundoff of the output type,
  |error| <= 6 u * scale * A  (conversions of acc and sum, the zero point's product, two scalings)
           + 2 u (|y| + |bias|) + v |y| + the output type's smallest step.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from stagehand_amd.int8 import Int8Tokens, Int8Weight, linear_i8, matmul_i8, quantize_tokens

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -149}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def np_quantize(x: np.ndarray):
    """(q, scale, sums) of float32 rows, in numpy's float32."""
    x = x.astype(np.float32)
    amax = np.abs(x).max(1)
    bad = ~np.isfinite(x).all(1)
    with np.errstate(all="ignore"):
        zero = amax < np.float32(2.0 ** -120)
        inv = np.where(bad | zero, np.float32(0), np.float32(127) / amax)
        scale = np.where(bad, np.float32("nan"), np.where(zero, np.float32(0), amax * (np.float32(1) / np.float32(127))))
        q = np.where((inv == 0)[:, None], np.float32(0), np.rint(x * inv[:, None]))
    q = q.astype(np.int8)
    return q, scale.astype(np.float32), q.astype(np.int64).sum(1)


def make(tokens, out, inp, *, pad=0, zp=False, bias=True, dtype=torch.bfloat16, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(tokens, inp, generator=g) * torch.exp(torch.randn(inp, generator=g))).to(dtype)
    q = torch.randint(-128, 128, (out, inp + pad), dtype=torch.int8, generator=g)
    s = torch.exp(torch.randn(out, generator=g) * 0.5 - 6)
    z = torch.randn(out, generator=g) * 3 if zp else None
    b = torch.randn(out, generator=g) if bias else None
    w = Int8Weight(q.cuda(), s.cuda(), None if z is None else z.cuda(), None if b is None else b.cuda(), inp)
    return x, q[:, :inp], s, z, b, w


def expect(x, q, s, z, b, dtype):
    """(y, tolerance) in float64."""
    tq, ts, sums = np_quantize(x.float().numpy())
    acc = (torch.from_numpy(tq).double() @ q.double().t()).numpy()
    y, size = acc, np.abs(acc)
    if z is not None:
        zs = z.numpy().astype(np.float64)[None] * sums[:, None]
        y, size = acc - zs, size + np.abs(zs)
    scale = ts.astype(np.float64)[:, None] * s.numpy().astype(np.float64)[None]
    y = y * scale
    bias = 0.0 if b is None else b.numpy().astype(np.float64)[None]
    y = y + bias
    tol = 6 * U * scale * size + 2 * U * (np.abs(y) + np.abs(bias)) + ROUND[dtype] * np.abs(y) + TINY[dtype]
    return y, tol


def check(got, x, q, s, z, b):
    y, tol = expect(x, q, s, z, b, got.dtype)
    got = got.reshape(y.shape).double().cpu().numpy()
    bad = ~(np.abs(got - y) <= tol)
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, first at {np.argwhere(bad)[0]}: {got[bad][0]} for {y[bad][0]}"


# ── quantisation ─────────────────────────────────────────────────────────────


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,cols", [(1, 1), (1, 4096), (3, 7), (5, 64), (70, 129), (257, 1155), (9, 8192), (4, 16384),
                                         (2, 40001), (33, 3072)])
def test_quantize_tokens_is_bit_exact(tokens, cols, dtype):
    g = torch.Generator().manual_seed(cols)
    x = (torch.randn(tokens, cols, generator=g) * torch.exp(2 * torch.randn(tokens, 1, generator=g))).to(dtype)
    t = quantize_tokens(x.cuda())
    q, scale, sums = np_quantize(x.float().numpy())
    assert t.q.shape == (tokens, -(-cols // 128) * 128) and t.in_features == cols and t.shape == (tokens,)
    got = t.q.cpu().numpy()
    np.testing.assert_array_equal(got[:, :cols], q)
    assert not got[:, cols:].any()
    np.testing.assert_array_equal(t.scale.cpu().numpy(), scale)
    np.testing.assert_array_equal(t.sums.cpu().numpy(), sums)


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_tokens_of_extreme_values(dtype):
    """Zeros, the smallest and largest magnitudes, infinities and NaNs: each token by itself."""
    big = torch.finfo(dtype).max
    rows = [[0.0] * 200, [1e-42] * 200, [2.0 ** -121] * 200, [2.0 ** -119, -(2.0 ** -120)] * 100, [big, -big] * 100,
            [1.0, float("inf")] + [2.0] * 198, [float("nan")] + [1.0] * 199, [0.0] * 199 + [float("-inf")],
            [1.0] * 199 + [float("nan")], [0.5, 1.0, -1.0, 0.25] * 50, [-0.0] * 200]
    x = torch.tensor(rows).to(dtype)
    t = quantize_tokens(x.cuda())
    q, scale, sums = np_quantize(x.float().numpy())
    np.testing.assert_array_equal(t.q.cpu().numpy()[:, :200], q)
    np.testing.assert_array_equal(t.scale.cpu().numpy(), scale)
    np.testing.assert_array_equal(t.sums.cpu().numpy(), sums)


def test_quantize_tokens_of_strided_and_offset_views():
    base = torch.randn(40, 3, 517, device="cuda", dtype=torch.bfloat16)
    for x in (base[:, 1], base[::3, 2, 5:400], base[:, 0, 1:], base.transpose(0, 1), base[..., ::2],
              base[0, 0], base[:1, :, :100].expand(6, 3, 100)):
        t = quantize_tokens(x)
        q, scale, sums = np_quantize(x.float().cpu().reshape(-1, x.shape[-1]).numpy())
        np.testing.assert_array_equal(t.q.cpu().numpy()[:, :x.shape[-1]], q)
        np.testing.assert_array_equal(t.scale.cpu().numpy(), scale)
        assert t.shape == x.shape[:-1] and t.dequantize().shape == x.shape


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [8, 9, 15, 203, 517, 2047])
def test_a_token_does_not_see_the_next_one(cols, dtype):
    """Ragged ends with infinities and NaNs right behind them, rows that overlap, and a last row that ends its memory."""
    x = torch.randn(12, cols).to(dtype)
    x[1::2, :8] = torch.tensor([float("inf"), float("nan"), float("-inf"), float("nan")] * 2)
    for v in (x.cuda(), x.cuda()[::2], x.cuda()[::2][:1].expand(5, cols), x.cuda().reshape(-1)[:cols * 8].as_strided((7, cols), (3, 1))):
        t = quantize_tokens(v)
        q, scale, sums = np_quantize(v.float().cpu().numpy())
        np.testing.assert_array_equal(t.q.cpu().numpy()[:, :cols], q)
        np.testing.assert_array_equal(t.scale.cpu().numpy(), scale)
        np.testing.assert_array_equal(t.sums.cpu().numpy(), sums)
        w = Int8Weight(torch.ones(3, cols, dtype=torch.int8, device="cuda"), torch.ones(3, device="cuda"))
        few = linear_i8(v, w).isnan().any(1).cpu().numpy()
        np.testing.assert_array_equal(few, np.isnan(scale))


# ── the product ──────────────────────────────────────────────────────────────

SIZES = [  # tokens, out, inp
    (1, 1, 1), (1, 64, 64), (1, 4096, 4096), (1, 999, 16384), (2, 130, 100), (3, 64, 1155), (4, 18432, 3072), (5, 256, 64),
    (7, 1000, 77), (8, 500, 2048), (15, 33, 129), (16, 1024, 1024), (17, 64, 65), (16, 31, 128), (31, 100, 1000),
    (32, 512, 512), (33, 257, 640), (64, 64, 4096), (65, 4096, 513), (77, 1000, 1155), (100, 1, 300), (127, 129, 127),
    (128, 128, 128), (129, 255, 384), (255, 257, 256), (256, 256, 256), (257, 513, 1025), (300, 1024, 96),
    (512, 1536, 512), (513, 320, 4097), (1024, 1024, 1024), (1025, 777, 130), (2048, 3072, 192), (4096, 64, 64),
    # ragged edges of the larger tiles, and columns of one, two and an odd number of 128-byte steps
    (1000, 2050, 300), (1023, 5000, 200), (2047, 4100, 130), (2049, 4097, 128), (4600, 3080, 257), (4609, 3071, 100),
    (3000, 6000, 640),
    # the most pieces of 512 values that one launch takes, and one more, for narrow and wide weights
    (8, 100, 4096), (9, 100, 4096), (16, 33, 2048), (15, 50, 2049), (1, 200, 32768), (1, 70, 32769), (16, 8161, 1024),
    (11, 8200, 1025), (1, 9000, 16384), (2, 8161, 8193), (16, 8160, 2000), (5, 20000, 513),
]


@pytest.mark.parametrize("tokens,out,inp", SIZES)
def test_linear_matches_64_bits(tokens, out, inp):
    seed = tokens * 31 + out
    x, q, s, z, b, w = make(tokens, out, inp, pad=(0, 3, 16)[seed % 3], zp=bool(seed & 1), bias=bool(seed & 2),
                            dtype=DTYPES[seed % 3], seed=seed)
    got = linear_i8(x.cuda(), w)
    assert got.dtype == x.dtype and got.shape == (tokens, out)
    check(got, x, q, s, z, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("zp", [False, True])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("tokens", [1, 6, 40, 200])
def test_linear_types_zero_points_and_bias(tokens, bias, zp, dtype):
    x, q, s, z, b, w = make(tokens, 320, 208, pad=5, zp=zp, bias=bias, dtype=dtype, seed=tokens)
    check(linear_i8(x.cuda(), w), x, q, s, z, b)


@pytest.mark.parametrize("out_dtype", DTYPES)
@pytest.mark.parametrize("tokens", [1, 50, 384])
def test_two_calls_equal_the_fused_one(tokens, out_dtype):
    x, q, s, z, b, w = make(tokens, 500, 700, zp=True, dtype=out_dtype, seed=3)
    t = quantize_tokens(x.cuda())
    y = matmul_i8(t, w, out_dtype=out_dtype)
    check(y, x, q, s, z, b)
    assert torch.equal(y, linear_i8(x.cuda(), w))


def test_extreme_products_do_not_overflow():
    """The largest count of columns with the largest magnitudes, of both signs."""
    cols = 131071
    x = torch.full((3, cols), 1.0)
    x[1] = -1.0
    x[2, ::2] = -1.0
    q = torch.full((4, cols), -128, dtype=torch.int8)
    q[1] = 127
    q[2, ::2] = 127
    s = torch.full((4,), 2.0 ** -10)
    w = Int8Weight(q.cuda(), s.cuda())
    check(linear_i8(x.cuda(), w), x, q, s, None, None)


@pytest.mark.parametrize("tokens", [5, 40, 300])
def test_nonfinite_tokens_stay_their_own(tokens):
    x, q, s, z, b, w = make(tokens, 130, 200, zp=True, dtype=torch.float32, seed=9)
    x[1, 7] = float("inf")
    x[3, 199] = float("nan")
    x[4] = 0
    y = linear_i8(x.cuda(), w).cpu()
    assert y[1].isnan().all() and y[3].isnan().all()
    assert torch.equal(y[4], b)
    keep = [i for i in range(tokens) if i not in (1, 3)]
    check(y[keep], x[keep], q, s, z, b)


def test_padding_columns_do_not_count():
    """Whatever lies between in_features and the row's end, and past the last row, is not read into the result."""
    for inp, ld in ((100, 112), (100, 160), (129, 144), (64, 80), (33, 48), (130, 256), (100, 128)):
        x, q, s, z, b, _ = make(9, 70, inp, zp=True, seed=inp)
        slab = torch.full((70, ld), 127, dtype=torch.int8, device="cuda")
        slab[:, :inp] = q.cuda()
        w = Int8Weight(slab, s.cuda(), z.cuda(), b.cuda(), inp, realign=ld % 128 == 0)
        assert w.qweight.data_ptr() == slab.data_ptr()
        check(linear_i8(x.cuda(), w), x, q, s, z, b)
        check(linear_i8(x.cuda().repeat(30, 1), w)[-9:], x, q, s, z, b)


def test_unaligned_weights_are_copied_once():
    x, q, s, z, b, _ = make(20, 50, 100, seed=1)
    flat = torch.zeros(50 * 100 + 1, dtype=torch.int8, device="cuda")
    flat[1:] = q.cuda().reshape(-1)
    for realign, ld in ((True, 128), (False, 112)):
        w = Int8Weight(flat[1:].view(50, 100), s.cuda(), bias=b.cuda(), realign=realign)
        assert w.qweight.stride(0) == ld and w.qweight.data_ptr() % 16 == 0
        check(linear_i8(x.cuda(), w), x, q, s, z, b)
    wide = torch.zeros(50, 144, dtype=torch.int8, device="cuda")
    wide[:, :100] = q.cuda()
    w = Int8Weight(wide, s.cuda(), bias=b.cuda(), in_features=100)
    assert w.qweight.stride(0) == 128
    check(linear_i8(x.cuda(), w), x, q, s, z, b)
    wt = Int8Weight(q.cuda().t().contiguous().t(), s.cuda(), bias=b.cuda())
    check(linear_i8(x.cuda(), wt), x, q, s, z, b)


def test_leading_dims_strides_and_out():
    x, q, s, z, b, w = make(24, 96, 160, zp=True, dtype=torch.float16, seed=5)
    want = linear_i8(x.cuda(), w)
    assert torch.equal(linear_i8(x.cuda().view(2, 3, 4, 160), w), want.view(2, 3, 4, 96))
    assert torch.equal(linear_i8(x.cuda()[0], w), want[0])
    wide = torch.zeros(24, 480, dtype=torch.float16, device="cuda")
    wide[:, 3:163] = x.cuda()
    assert torch.equal(linear_i8(wide[:, 3:163], w), want)
    assert torch.equal(linear_i8(x.cuda().t().contiguous().t(), w), want)
    out = torch.full((24, 200), 7.0, dtype=torch.float16, device="cuda")
    got = linear_i8(x.cuda(), w, out=out[:, 101:197])
    assert got.data_ptr() == out[:, 101:197].data_ptr()
    assert torch.equal(out[:, 101:197], want) and bool((out[:, :101] == 7).all()) and bool((out[:, 197:] == 7).all())
    big = torch.full((300, 131), 5.0, dtype=torch.float16, device="cuda")
    xs = x.cuda().repeat(12, 1)
    linear_i8(xs, w, out=big[:288, 1:97])
    assert torch.equal(big[:288, 1:97], want.repeat(12, 1))
    assert bool((big[288:] == 5).all()) and bool((big[:, 0] == 5).all()) and bool((big[:, 97:] == 5).all())


def test_no_tokens_and_no_rows():
    _, _, s, _, _, w = make(2, 40, 30)
    assert linear_i8(torch.empty(0, 30, device="cuda"), w).shape == (0, 40)
    assert linear_i8(torch.empty(3, 0, 30, device="cuda"), w).shape == (3, 0, 40)
    assert quantize_tokens(torch.empty(0, 30, device="cuda")).q.shape == (0, 128)
    w0 = Int8Weight(torch.empty(0, 30, dtype=torch.int8, device="cuda"), torch.empty(0, device="cuda"))
    assert linear_i8(torch.ones(5, 30, device="cuda"), w0).shape == (5, 0)


@pytest.mark.parametrize("tokens", [4, 200])
def test_another_stream_and_a_captured_graph(tokens):
    x, q, s, z, b, w = make(tokens, 300, 520, zp=True, seed=2)
    x = x.cuda()
    want = linear_i8(x, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    y = linear_i8(x, w, stream=side)
    side.synchronize()
    assert torch.equal(y, want)
    assert torch.equal(linear_i8(x, w, stream=torch.cuda.current_stream().cuda_stream), want)
    graph = torch.cuda.CUDAGraph()
    fixed = x.clone()
    with torch.cuda.graph(graph):
        y = linear_i8(fixed, w)
    for k in range(3):
        fixed.copy_(x * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, linear_i8(x * (k + 1), w))


def test_repeated_calls_give_the_same_bits():
    for tokens in (1, 12, 60, 700):
        x, q, s, z, b, w = make(tokens, 1024, 2048, zp=True, seed=tokens)
        x = x.cuda()
        first = linear_i8(x, w)
        for _ in range(5):
            assert torch.equal(linear_i8(x, w), first)


def test_offsets_past_32_bits():
    """Tokens and outputs whose places pass 2^32 elements, and a weight of more than 4 GiB."""
    cols, tokens = 131008, 40000
    x = torch.zeros(tokens, cols, dtype=torch.bfloat16, device="cuda")
    tail = torch.randn(3, cols).to(torch.bfloat16)
    x[-3:] = tail.cuda()
    q = torch.randint(-128, 128, (50, cols), dtype=torch.int8)
    s = torch.full((50,), 0.01)
    w = Int8Weight(q.cuda(), s.cuda())
    y = linear_i8(x, w)
    check(y[-3:], tail, q, s, None, None)
    assert not bool(y[:-3].any())
    del x, y
    rows = 33000
    big = torch.zeros(rows, cols, dtype=torch.int8, device="cuda")
    big[-50:] = q.cuda()
    wb = Int8Weight(big, torch.full((rows,), 0.01, device="cuda"))
    for n in (1, 3, 40):
        xt = tail[:1].repeat(n, 1) if n != 3 else tail
        y = linear_i8(xt.cuda(), wb)
        check(y[:, -50:], xt, q, s, None, None)
        assert not bool(y[:, :-50].any())
    del big, wb, y
    wide = Int8Weight(q[:, :64].contiguous().cuda().repeat(1400, 1), torch.full((70000,), 0.01, device="cuda"))
    xs = torch.randn(62000, 64).to(torch.bfloat16)
    y = linear_i8(xs.cuda(), wide)  # 4.3 G outputs
    check(y[-300:, -50:], xs[-300:], q[:, :64], s, None, None)
    check(y[:300, :50], xs[:300], q[:, :64], s, None, None)


def test_squareq_layers(tmp_path):
    from stagehand_amd.squareq_v2 import read_v2_layers, write_v2_slab

    g = torch.Generator().manual_seed(0)
    layer = {"qweight": torch.randint(-127, 128, (96, 80), dtype=torch.int8, generator=g),
             "scale": torch.rand(96, generator=g) * 0.01, "zero_point": torch.randn(96, generator=g),
             "bias": torch.randn(96, generator=g).to(torch.bfloat16), "in_features": 77}
    path = str(tmp_path / "slab.safetensors")
    manifest = write_v2_slab(path, {"fc": layer, "plain": {k: layer[k].clone() for k in ("qweight", "scale")}})
    view = memoryview(bytearray(open(path, "rb").read()))
    layers = read_v2_layers(path, manifest, view)
    w = Int8Weight.from_squareq(layers["fc"], 96, 77)
    x = torch.randn(19, 77).to(torch.bfloat16)
    check(linear_i8(x.cuda(), w), x, layer["qweight"][:, :77], layer["scale"], layer["zero_point"], layer["bias"].float())
    plain = Int8Weight.from_squareq(layers["plain"], 96, 77)
    assert plain.zero_point is None and plain.bias is None
    want = (layer["qweight"][:, :77].float() - layer["zero_point"][:, None]) * layer["scale"][:, None]
    assert torch.equal(w.dequantize(torch.bfloat16).cpu(), want.to(torch.bfloat16))


# ── refusals ─────────────────────────────────────────────────────────────────


def test_refusals():
    _, q, s, z, b, w = make(4, 40, 32)
    x = torch.randn(4, 32, device="cuda")
    bad = [
        lambda: linear_i8(x[:, :31], w), lambda: linear_i8(x.double(), w), lambda: linear_i8(x.int(), w),
        lambda: linear_i8(x.cpu(), w), lambda: linear_i8(torch.tensor(1.0, device="cuda"), w),
        lambda: linear_i8(x, w, out=torch.empty(4, 41, device="cuda")),
        lambda: linear_i8(x, w, out=torch.empty(4, 40, device="cuda", dtype=torch.bfloat16)),
        lambda: linear_i8(x, w, out=torch.empty(40, 4, device="cuda").t()),
        lambda: linear_i8(x, w, out=torch.empty(4, 40)),
        lambda: linear_i8(x, w, out=torch.empty(1, 40, device="cuda").expand(4, 40)),
        lambda: quantize_tokens(torch.empty(2, 0, device="cuda")),
        lambda: quantize_tokens(torch.empty(2, 131072, device="cuda")),
        lambda: matmul_i8(quantize_tokens(x[:, :16]), w), lambda: matmul_i8(quantize_tokens(x), w, out_dtype=torch.float64),
        lambda: matmul_i8(quantize_tokens(x)._replace(q=x), w),
        lambda: matmul_i8(quantize_tokens(x)._replace(scale=torch.ones(3, device="cuda")), w),
        lambda: matmul_i8(quantize_tokens(x)._replace(shape=torch.Size((5,))), w),
        lambda: matmul_i8(Int8Tokens(torch.zeros(4, 32, dtype=torch.int8, device="cuda"), torch.ones(4, device="cuda"),
                                     torch.ones(4, dtype=torch.int32, device="cuda"), 32, torch.Size((4,))), w),
        lambda: Int8Weight(q.cuda().float(), s.cuda()), lambda: Int8Weight(q, s),
        lambda: Int8Weight(q.cuda()[0], s.cuda()), lambda: Int8Weight(q.cuda(), s.cuda()[1:]),
        lambda: Int8Weight(q.cuda(), s.cuda(), zero_point=s.cuda()[1:]), lambda: Int8Weight(q.cuda(), s.cuda(), in_features=33),
        lambda: Int8Weight(q.cuda(), s.cuda(), in_features=0), lambda: Int8Weight(q.cuda(), s.cuda().int()),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    with pytest.raises(RuntimeError, match="no gradient"):
        linear_i8(x.clone().requires_grad_(), w)
    with torch.no_grad():
        linear_i8(x.clone().requires_grad_(), w)
