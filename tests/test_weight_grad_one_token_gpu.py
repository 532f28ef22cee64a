"""The weight gradient's C entry: with one token there is no distance between rows, whatever is given for it."""
from __future__ import annotations

import ctypes

import pytest
import torch
from act8_oracle import DTYPES

from stagehand_amd import _native, act8
from stagehand_amd.int8 import DTYPE_CODES
from stagehand_amd.unpack import current_stream_handle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("out", [1, 8, 33, 300])
def test_one_token(out, dtype):
    g = torch.Generator(device="cuda").manual_seed(out)
    x = (0.5 + torch.rand(1, 70, device="cuda", generator=g)).to(dtype)  # none is kept as 0
    dy = torch.randn(1, out, device="cuda", generator=g).to(dtype)
    dy[0, out // 2] = float("inf")
    kept = act8.quantize_activation(x)
    args, _ = act8._kept_args(kept)
    lib, need, code = _native.lib(), ctypes.c_uint64(), DTYPE_CODES[dtype]
    _native.check(lib.sh_weight_grad_act8_workspace(args, code, out, True, ctypes.byref(need)))
    assert need.value == 0  # a token is not split
    want = dy.double().t().contiguous() * kept.dequantize().double()
    for ld in (out, 0, 1, out - 1, act8.MAX_OUT):
        dw, db = torch.empty(out, 70, device="cuda"), torch.empty(out, device="cuda")
        _native.check(lib.sh_weight_grad_act8(dy.data_ptr(), code, ld, out, args, dw.data_ptr(), 3, 70, db.data_ptr(), None, 0, current_stream_handle()))
        assert torch.equal(db, dy[0].float()), ld
        # one product: exact in 16 bits; three, of parts of 8 bits each, in 32
        finite = want.isfinite()
        assert torch.equal(finite, dw.isfinite()) and torch.equal(dw[~finite], want[~finite].float()), ld
        assert bool(((dw.double() - want)[finite].abs() <= 3 * 2.0 ** -24 * want[finite].abs()).all()), ld
