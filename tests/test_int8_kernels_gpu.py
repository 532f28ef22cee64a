"""Int8 linear layers at sizes for each kernel: every tile of the product and every one-launch kernel, in each type,
with and without zero points and bias. test_operator_dispatch says which kernel a size takes. Tolerances as in
test_int8_gpu."""
from __future__ import annotations

import pytest
from test_int8_gpu import DTYPES, check, make

from stagehand_amd.int8 import linear_i8

pytestmark = pytest.mark.gpu

# 128 x 128 tiles: whole, ragged in tokens, rows and columns, one and two steps of columns, many tiles
TILE_128 = [(256, 9216, 256), (250, 9200, 300), (1024, 4096, 130), (240, 9100, 100), (384, 8200, 384)]
# one launch, for wide and for narrow weights: one token, some, sixteen, ragged ends
FEW_WIDE = [(1, 8200, 3000), (4, 9000, 3072), (16, 8161, 1024), (5, 20000, 513), (3, 8200, 77)]
FEW_NARROW = [(1, 4096, 4096), (7, 1000, 1100), (16, 8160, 700), (2, 31, 16000), (12, 500, 40)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("zp,bias", [(False, True), (True, False), (True, True), (False, False)])
@pytest.mark.parametrize("tokens,out,inp", TILE_128 + FEW_WIDE + FEW_NARROW)
def test_every_kernel_in_every_type(tokens, out, inp, zp, bias, dtype):
    x, q, s, z, b, w = make(tokens, out, inp, pad=(0, 3)[tokens % 2], zp=zp, bias=bias, dtype=dtype, seed=out)
    check(linear_i8(x.cuda(), w), x, q, s, z, b)
