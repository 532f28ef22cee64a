"""Products of tokens whose rows are some of a larger tensor's: every second token, the last of each sequence,
columns of wider rows, rows that end with their memory. Only a token's own columns count, however far apart the
tokens lie. Tolerances as in test_int8_gpu."""
from __future__ import annotations

import pytest
import torch
from test_int8_gpu import check, make

from stagehand_amd.int8 import Int8Tokens, matmul_i8, quantize_tokens

pytestmark = pytest.mark.gpu

# tokens, out, inp: each tile of the product, one and several steps of 128 columns, ragged and whole ends
SIZES = [(1, 40, 100), (3, 50, 128), (9, 130, 300), (20, 9000, 200), (40, 257, 385), (100, 900, 130), (250, 9200, 100),
         (600, 4100, 140), (1100, 8200, 260)]


def quantised(tokens, out, inp, zp=True):
    x, q, s, z, b, w = make(tokens, out, inp, zp=zp, seed=tokens + inp)
    return quantize_tokens(x.cuda()), w, (x, q, s, z, b)


def laid_out(t: Int8Tokens, q: torch.Tensor) -> Int8Tokens:
    assert torch.equal(q[:, :t.q.shape[1]], t.q)
    return t._replace(q=q)


@pytest.mark.parametrize("tokens,out,inp", SIZES)
def test_columns_of_wider_rows(tokens, out, inp):
    """What lies beside a token's columns is not read, whether it comes before, behind or not at all."""
    t, w, ref = quantised(tokens, out, inp)
    width = t.q.shape[1]
    for before, behind in ((0, 128), (128, 0), (256, 384)):
        wide = torch.full((tokens, before + width + behind), 77, dtype=torch.int8, device="cuda")
        wide[:, before:before + width] = t.q
        check(matmul_i8(laid_out(t, wide[:, before:before + width]), w, out_dtype=torch.float32), *ref)
        if behind:
            check(matmul_i8(laid_out(t, wide[:, before:]), w, out_dtype=torch.float32), *ref)


@pytest.mark.parametrize("tokens,out,inp", SIZES)
def test_every_second_token_and_the_last_of_each_sequence(tokens, out, inp):
    t, w, ref = quantised(tokens, out, inp)
    for step, at in ((2, 0), (3, 2)):
        many = torch.full((tokens, step, t.q.shape[1]), -99, dtype=torch.int8, device="cuda")
        many[:, at] = t.q
        picked = many[:, at]
        check(matmul_i8(laid_out(t, picked), w, out_dtype=torch.float32), *ref)
        flat = many.view(tokens * step, -1)[at::step]
        check(matmul_i8(laid_out(t, flat), w, out_dtype=torch.float32), *ref)


@pytest.mark.parametrize("tokens,out,inp", SIZES)
def test_rows_that_end_with_their_memory(tokens, out, inp):
    """The last row is followed by nothing: its memory ends where its columns do."""
    t, w, ref = quantised(tokens, out, inp)
    width = t.q.shape[1]
    ld = width + 256
    flat = torch.full(((tokens - 1) * ld + width,), 55, dtype=torch.int8, device="cuda")
    view = flat.as_strided((tokens, width), (ld, 1))
    view.copy_(t.q)
    check(matmul_i8(laid_out(t, view), w, out_dtype=torch.float32), *ref)


@pytest.mark.parametrize("tokens,out,inp", SIZES)
def test_rows_that_cannot_be_read_in_place(tokens, out, inp):
    """Rows off 128-byte distances or 16-byte boundaries, rows further apart than a product's offsets reach, one
    row for all tokens."""
    t, w, ref = quantised(tokens, out, inp)
    width = t.q.shape[1]
    for before, behind in ((0, 24), (5, 0), (1, 127)):
        wide = torch.full((tokens, before + width + behind), 31, dtype=torch.int8, device="cuda")
        wide[:, before:before + width] = t.q
        check(matmul_i8(laid_out(t, wide[:, before:before + width]), w, out_dtype=torch.float32), *ref)
    far = torch.empty(tokens, (1 << 20) + 128, dtype=torch.int8, device="cuda")
    far[:, :width] = t.q
    check(matmul_i8(laid_out(t, far[:, :width]), w, out_dtype=torch.float32), *ref)
    same = Int8Tokens(t.q[:1].expand(tokens, width), t.scale[:1].repeat(tokens), t.sums[:1].repeat(tokens), inp, t.shape)
    y = matmul_i8(same, w, out_dtype=torch.float32)
    assert torch.equal(y, matmul_i8(same._replace(q=same.q.contiguous()), w, out_dtype=torch.float32))
    check(y[:1], ref[0][:1], *ref[1:])


def test_rows_shorter_than_a_token_are_refused():
    t, w, _ = quantised(6, 40, 100)
    with pytest.raises(ValueError, match="zeros up to 128"):
        matmul_i8(t._replace(q=t.q[:, :100]), w)
    with pytest.raises(ValueError, match="zeros up to 128"):
        matmul_i8(t._replace(q=t.q[:, :112].contiguous()), w)
