"""Int8 linear layers at the ends of their ranges: token scales from 2^-127 to the type's largest, integer zero
points, counts past 32 bits. Tolerances as in test_int8_gpu."""
from __future__ import annotations

import pytest
import torch
from test_int8_gpu import check, make

from stagehand_amd.int8 import Int8Weight, linear_i8, matmul_i8, quantize_tokens

pytestmark = pytest.mark.gpu

# tokens, out, inp: one launch, two with few tokens, and the tiles
SIZES = [(3, 100, 200), (5, 9000, 300), (24, 9000, 100), (40, 100, 130), (100, 900, 200), (250, 9200, 130), (600, 4100, 140),
         (1100, 8200, 260)]


def scaled(tokens, out, inp, dtype, zp, exponents, row_exponents):
    """Tokens and rows whose magnitudes are spread evenly over the exponents given."""
    x, q, _, z, _, _ = make(tokens, out, inp, zp=zp, bias=False, dtype=torch.float32, seed=tokens)
    g = torch.Generator().manual_seed(1)
    e = torch.linspace(*exponents, tokens).round()[torch.randperm(tokens, generator=g)]
    x = x / x.abs().amax(1, keepdim=True)  # largest magnitude 1
    x = (x.double() * torch.exp2(e.double())[:, None]).float().to(dtype)
    r = torch.linspace(*row_exponents, out).round()[torch.randperm(out, generator=g)]
    s = ((1 + torch.rand(out, generator=g).double()) * torch.exp2(r.double())).float()
    return x, q, s, z, None, Int8Weight(q.cuda(), s.cuda(), None if z is None else z.cuda(), None, inp)


@pytest.mark.parametrize("zp", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens,out,inp", SIZES)
@pytest.mark.parametrize("exponents,row_exponents", [((-119, -100), (-20, 0)), ((100, 127), (-60, -40)), ((-119, 127), (-30, -30)),
                                                     ((-119, -119), (40, 60))])
def test_token_scales_of_any_size(tokens, out, inp, dtype, zp, exponents, row_exponents):
    x, q, s, z, b, w = scaled(tokens, out, inp, dtype, zp, exponents, row_exponents)
    got = linear_i8(x.cuda(), w)
    check(got, x, q, s, z, b)
    assert torch.equal(got, matmul_i8(quantize_tokens(x.cuda()), w, out_dtype=dtype))


@pytest.mark.parametrize("tokens", [3, 40, 300])
def test_a_sum_of_zero_is_zero_whatever_its_scales(tokens):
    """Scales whose product overflows, where the integers cancel: the bias, not NaN."""
    x = torch.full((tokens, 64), 3e38)
    x[:, ::2] = -3e38
    b = torch.randn(70)
    w = Int8Weight(torch.full((70, 64), 5, dtype=torch.int8, device="cuda"), torch.full((70,), 1e10, device="cuda"), bias=b.cuda())
    assert torch.equal(linear_i8(x.cuda(), w).cpu(), b.expand(tokens, 70))


def test_integer_zero_points():
    """A slab may hold its zero points as integers; the dequantising path takes them too."""
    x, q, s, _, b, _ = make(20, 50, 90, seed=4)
    z = torch.randint(-100, 100, (50,))
    for zdt in (torch.int8, torch.int16, torch.int32, torch.int64):
        zi = z.to(zdt)
        w = Int8Weight(q.cuda(), s.cuda(), zi.cuda(), b.cuda())
        check(linear_i8(x.cuda(), w), x, q, s, z.float(), b)
        ws = Int8Weight.from_squareq({"qweight": q, "scale": s, "zero_point": zi, "bias": b})
        assert torch.equal(linear_i8(x.cuda(), ws), linear_i8(x.cuda(), w))
    wu = Int8Weight(q.cuda(), s.cuda(), (z + 100).to(torch.uint8).cuda(), b.cuda())
    check(linear_i8(x.cuda(), wu), x, q, s, (z + 100).float(), b)
    for wrong in (torch.ones(50, dtype=torch.bool), torch.ones(50, dtype=torch.complex64)):
        with pytest.raises(ValueError, match="zero_point"):
            Int8Weight(q.cuda(), s.cuda(), wrong.cuda())


def test_counts_past_32_bits_are_refused():
    """2^32 + 3 tokens (one value seen that often) are not taken for three."""
    many = 2 ** 32 + 3
    w = Int8Weight(torch.ones(1, 8, dtype=torch.int8, device="cuda"), torch.ones(1, device="cuda"))
    x = torch.ones(1, 8, device="cuda", dtype=torch.bfloat16).expand(many, 8)
    with pytest.raises(ValueError, match="tokens"):
        linear_i8(x, w)
    with pytest.raises(ValueError, match="tokens"):
        quantize_tokens(x)
    with pytest.raises(ValueError, match="rows"):
        Int8Weight(torch.ones(1, 8, dtype=torch.int8, device="cuda").expand(many, 8), torch.ones(1, device="cuda").expand(many))
