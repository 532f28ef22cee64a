"""The operators' C entry points refuse what their kernels cannot take, before any GPU call (CPU only), and the
Python mirrors of their structs have the C layout."""
from __future__ import annotations

import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest

from stagehand_amd import _native, int8, qk_norm

HEADER = Path(__file__).resolve().parent.parent / "include" / "stagehand_native.h"
P = 1 << 20  # an aligned address that no refused call reads

QK_FIELDS = [f"{h}.{f}" for h in ("q", "k", "q_out", "k_out", "dq", "dk")
             for f in ("data", "batch_stride", "head_stride", "seq_stride")] + [
    "q_weight", "k_weight", "dq_weight", "dk_weight", "cos", "sin", "positions", "table_ld", "position_batch_stride", "start",
    "table_rows", "position_bytes", "batch", "seq", "q_heads", "k_heads", "dim", "rot", "dtype", "weight_dtype",
    "interleaved", "eps"]


def refused(name, *args, match):
    st = getattr(_native.lib(), name)(*args)
    assert st == _native.SH_ERR_INVALID, (name, st, _native.last_error())
    assert name in _native.last_error() and match in _native.last_error(), _native.last_error()


def weight(**kw):
    w = dict(q=P, ld=64, rows=8, cols=64, scale=P, zero_point=0, bias=0)
    w.update(kw)
    return ctypes.byref(int8._Weight(*w.values()))


def test_struct_mirrors_match_the_c_layout(tmp_path):
    if shutil.which("gcc") is None:
        pytest.skip("gcc is not available")
    w = [n for n, _ in int8._Weight._fields_]
    src = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {",
           'printf("%zu %zu\\n", sizeof(sh_i8_weight), sizeof(sh_qk_norm_rope_args));']
    src += [f'printf("%zu\\n", offsetof(sh_i8_weight, {n}));' for n in w]
    src += [f'printf("%zu\\n", offsetof(sh_qk_norm_rope_args, {n}));' for n in QK_FIELDS]
    src += ['printf("%u %u %u\\n", SH_I8_MAX_COLS, SH_I8_TOKEN_ALIGN, SH_QK_MAX_DIM);', "return 0; }"]
    (tmp_path / "a.c").write_text("\n".join(src))
    subprocess.run(["gcc", str(tmp_path / "a.c"), "-o", str(tmp_path / "a")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "a")], check=True, capture_output=True, text=True).stdout.split()]
    assert got[:2] == [ctypes.sizeof(int8._Weight), qk_norm._ARGS.size]
    assert got[2:2 + len(w)] == [getattr(int8._Weight, n).offset for n in w]
    sizes = [8] * 34 + [4] * 12
    assert got[2 + len(w):-3] == [sum(sizes[:i]) for i in range(len(QK_FIELDS))]
    assert got[-3:] == [int8.MAX_COLS, int8.TOKEN_ALIGN, qk_norm.MAX_DIM]


def test_quantize_tokens_refusals():
    call = ("sh_quantize_tokens",)
    ok = dict(x=P, dtype=1, x_ld=64, tokens=2, cols=64, q=P, q_ld=128, scale=P, sums=0, stream=0)

    def bad(match, **kw):
        refused(*call, *{**ok, **kw}.values(), match=match)

    bad("dtype", dtype=0)
    bad("dtype", dtype=9)
    bad("cols", cols=0)
    bad("cols", cols=131072)
    bad("x is NULL", x=0)
    bad("aligned", x=P + 1)
    bad("q_ld", q_ld=64)
    bad("q_ld", q_ld=129)
    bad("q_ld", cols=200)
    bad("NULL", q=0)
    bad("NULL", scale=0)
    bad("aligned", q=P + 8)
    bad("aligned", scale=P + 2)
    bad("aligned", sums=P + 1)
    bad("too many", tokens=0xFFFFFFFF)
    assert _native.lib().sh_quantize_tokens(*{**ok, "tokens": 0, "x": 0, "q": 0, "scale": 0}.values()) == _native.SH_OK


def test_matmul_and_linear_refusals():
    ok = dict(q=P, q_ld=128, scale=P, sums=P, tokens=2, w=weight(), out=P, out_dtype=1, out_ld=8, stream=0)

    def bad(match, **kw):
        refused("sh_matmul_i8", *{**ok, **kw}.values(), match=match)

    bad("w is NULL", w=None)
    bad("cols", w=weight(cols=0))
    bad("cols", w=weight(cols=200000, ld=200000))
    bad("ld", w=weight(ld=72))
    bad("ld", w=weight(ld=48))
    bad("ld", w=weight(ld=1 << 21))
    bad("NULL", w=weight(q=0))
    bad("NULL", w=weight(scale=0))
    bad("aligned", w=weight(q=P + 4))
    bad("aligned", w=weight(scale=P + 2))
    bad("aligned", w=weight(zero_point=P + 2))
    bad("aligned", w=weight(bias=P + 1))
    bad("q_ld", q_ld=64)
    bad("NULL", q=0)
    bad("NULL", scale=0)
    bad("sums is NULL", sums=0, w=weight(zero_point=P))
    bad("out dtype", out_dtype=4)
    bad("out is NULL", out=0)
    bad("aligned", out=P + 1)
    bad("out_ld", out_ld=7)
    bad("too many", tokens=0xFFFFFFFF, w=weight(rows=0xFFFFFFFF), out_ld=0xFFFFFFFF)
    assert _native.lib().sh_matmul_i8(*{**ok, "tokens": 0}.values()) == _native.SH_OK

    need = ctypes.c_uint64()
    refused("sh_linear_i8_workspace", 3, weight(), None, match="NULL")
    refused("sh_linear_i8_workspace", 3, None, ctypes.byref(need), match="NULL")
    refused("sh_linear_i8_workspace", 3, weight(ld=72), ctypes.byref(need), match="ld")
    assert _native.lib().sh_linear_i8_workspace(1, weight(), ctypes.byref(need)) == _native.SH_OK and need.value == 0
    assert _native.lib().sh_linear_i8_workspace(1000, weight(), ctypes.byref(need)) == _native.SH_OK
    assert need.value >= 1000 * (128 + 8)
    ok = dict(x=P, dtype=1, x_ld=64, tokens=1000, w=weight(), out=P, out_ld=8, ws=P, ws_bytes=need.value, stream=0)

    def bad_linear(match, **kw):
        refused("sh_linear_i8", *{**ok, **kw}.values(), match=match)

    bad_linear("dtype", dtype=5)
    bad_linear("w is NULL", w=None)
    bad_linear("x is NULL", x=0)
    bad_linear("aligned", x=P + 1)
    bad_linear("out is NULL", out=0)
    bad_linear("out_ld", out_ld=1)
    bad_linear("workspace", ws=0)
    bad_linear("workspace", ws_bytes=need.value - 1)
    bad_linear("workspace", ws=P + 8)
    assert _native.lib().sh_linear_i8(*{**ok, "tokens": 0, "ws": 0, "ws_bytes": 0}.values()) == _native.SH_OK


def test_qk_norm_refusals():
    ok = dict.fromkeys(QK_FIELDS, 0)
    for h in ("q", "k", "q_out", "k_out", "dq", "dk"):
        ok[f"{h}.data"] = P
    ok.update(cos=P, sin=P, table_ld=32, table_rows=16, position_bytes=8, batch=1, seq=4, q_heads=2, k_heads=1, dim=64, rot=64,
              dtype=1, weight_dtype=3, eps=1e-6)

    def bad(match, backward=False, **kw):
        args = qk_norm._ARGS.pack(*{**ok, **{k.replace("__", "."): v for k, v in kw.items()}}.values())
        refused("sh_qk_norm_rope_backward", args, P, 1 << 30, 0, match=match)
        if not backward:
            refused("sh_qk_norm_rope", args, 0, match=match)

    refused("sh_qk_norm_rope", None, 0, match="NULL")
    refused("sh_qk_norm_rope_backward", None, P, 1 << 30, 0, match="NULL")
    refused("sh_qk_norm_rope_workspace", None, ctypes.byref(ctypes.c_uint64()), match="NULL")
    bad("dtype", dtype=0)
    bad("weight_dtype", weight_dtype=7)
    for dim in (0, 1, 63, 514):
        bad("dim", dim=dim, rot=0)
    bad("rot", rot=66)
    bad("rot", rot=33)
    bad("eps", eps=-1e-9)
    bad("eps", eps=float("inf"))
    bad("eps", eps=float("nan"))
    bad("too many", batch=1 << 20, seq=1 << 20)
    bad("NULL", cos=0)
    bad("NULL", sin=0)
    bad("aligned", cos=P + 2)
    bad("table_ld", table_ld=31)
    bad("position_bytes", positions=P, position_bytes=2)
    bad("aligned", positions=P + 4)
    bad("tables", start=13)
    bad("tables", start=-1)
    bad("tables", start=1 << 40)
    bad("q is NULL", q__data=0)
    bad("k_out is NULL", k_out__data=0)
    bad("aligned", q_out__data=P + 1)
    bad("aligned", q_weight=P + 2)
    bad("aligned", backward=True, dq__data=P + 1)
    bad("aligned", backward=True, dk_weight=P + 1)
    args = qk_norm._ARGS.pack(*{**ok, "dq_weight": P}.values())
    need = ctypes.c_uint64()
    refused("sh_qk_norm_rope_workspace", args, None, match="NULL")
    assert _native.lib().sh_qk_norm_rope_workspace(args, ctypes.byref(need)) == _native.SH_OK and need.value > 0
    refused("sh_qk_norm_rope_backward", args, P, need.value - 1, 0, match="workspace")
    refused("sh_qk_norm_rope_backward", args, 0, need.value, 0, match="workspace")
    refused("sh_qk_norm_rope_backward", args, P + 4, need.value, 0, match="aligned")
    nothing = qk_norm._ARGS.pack(*{**ok, "batch": 0}.values())
    assert _native.lib().sh_qk_norm_rope(nothing, 0) == _native.SH_OK
    assert _native.lib().sh_qk_norm_rope_backward(nothing, 0, 0, 0) == _native.SH_OK
