"""The training operators' C entry points refuse what their kernels cannot take, before any GPU call (CPU only), the
Python mirrors of their structs have the C layout, and their streams are taken on the tensors' device."""
from __future__ import annotations

import ctypes
import shutil
import subprocess
from contextlib import nullcontext
from pathlib import Path
from types import SimpleNamespace

import pytest
import torch

from stagehand_amd import _native, act8, layer_norm

HEADER = Path(__file__).resolve().parent.parent / "include" / "stagehand_native.h"
P = 1 << 20  # an aligned address that no refused call reads

NORM_FIELDS = [f"{r}.{f}" for r in ("x", "y", "dy", "dx") for f in ("data", "batch_stride", "seq_stride")] + [
    "weight", "bias", "dweight", "dbias", "stats", "q", "exponent", "weight_batch_stride", "bias_batch_stride", "batch", "seq", "cols",
    "dtype", "weight_dtype", "per_batch", "modulate", "eps"]


def refused(name, *args, match):
    st = getattr(_native.lib(), name)(*args)
    assert st == _native.SH_ERR_INVALID, (name, st, _native.last_error())
    assert name in _native.last_error() and match in _native.last_error(), _native.last_error()


def kept(**kw):
    return act8._KEPT.pack(*{**dict(q=P, exponent=P, tokens=8, cols=64), **kw}.values())


def test_struct_mirrors_match_the_c_layout(tmp_path):
    if shutil.which("gcc") is None:
        pytest.skip("gcc is not available")
    src = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {",
           'printf("%zu %zu\\n", sizeof(sh_act8), sizeof(sh_layer_norm_args));']
    src += [f'printf("%zu\\n", offsetof(sh_act8, {n}));' for n in ("q", "exponent", "tokens", "cols")]
    src += [f'printf("%zu\\n", offsetof(sh_layer_norm_args, {n}));' for n in NORM_FIELDS]
    src += ['printf("%u %u %u %u\\n", SH_ACT8_GROUP, SH_ACT8_MAX_COLS, SH_WEIGHT_GRAD_MAX_OUT, SH_LAYER_NORM_MAX_COLS);', "return 0; }"]
    (tmp_path / "a.c").write_text("\n".join(src))
    subprocess.run(["gcc", str(tmp_path / "a.c"), "-o", str(tmp_path / "a")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "a")], check=True, capture_output=True, text=True).stdout.split()]
    assert got[:2] == [act8._KEPT.size, layer_norm._ARGS.size]
    assert got[2:6] == [0, 8, 16, 20]
    sizes = [8] * 21 + [4] * 8
    assert got[6:-4] == [sum(sizes[:i]) for i in range(len(NORM_FIELDS))]
    assert got[-4:] == [act8.GROUP, act8.MAX_COLS, act8.MAX_OUT, layer_norm.MAX_COLS] and layer_norm.GROUP == act8.GROUP


def test_act8_refusals():
    for name, order in (("sh_act8_quantize", ("x", "dtype", "ld", "kept", "stream")), ("sh_act8_dequantize", ("kept", "x", "dtype", "ld", "stream"))):
        ok = dict(x=P, dtype=1, ld=64, kept=kept(), stream=0)

        def bad(match, **kw):
            refused(name, *[{**ok, **kw}[k] for k in order], match=match)

        bad("kept is NULL", kept=None)
        bad("cols", kept=kept(cols=0))
        bad("cols", kept=kept(cols=1 << 24))
        bad("too many", kept=kept(tokens=1 << 30, cols=64))
        bad("NULL", kept=kept(q=0))
        bad("NULL", kept=kept(exponent=0))
        bad("aligned", kept=kept(q=P + 8))
        bad("dtype", dtype=0)
        bad("dtype", dtype=4)
        bad("NULL", x=0)
        bad("aligned", x=P + 1)
        if name == "sh_act8_dequantize":
            bad("out_ld", ld=63)
        assert getattr(_native.lib(), name)(*[{**ok, "kept": kept(tokens=0, q=0, exponent=0), "x": 0}[k] for k in order]) == _native.SH_OK


def test_weight_grad_refusals():
    need = ctypes.c_uint64()
    assert _native.lib().sh_weight_grad_act8_workspace(kept(tokens=4096), 1, 32, 1, ctypes.byref(need)) == _native.SH_OK
    assert need.value >= 4 * 2 * (32 * 64 + 32) and need.value % 4 == 0
    refused("sh_weight_grad_act8_workspace", kept(), 1, 32, 1, None, match="NULL")
    refused("sh_weight_grad_act8_workspace", None, 1, 32, 1, ctypes.byref(need), match="NULL")
    refused("sh_weight_grad_act8_workspace", kept(), 7, 32, 1, ctypes.byref(need), match="dtype")
    refused("sh_weight_grad_act8_workspace", kept(cols=0), 1, 32, 1, ctypes.byref(need), match="cols")
    ok = dict(dy=P, dtype=1, dy_ld=32, out=32, kept=kept(tokens=4096), dweight=P, out_dtype=3, dw_ld=64, dbias=P, ws=P, ws_bytes=need.value,
              stream=0)

    def bad(match, **kw):
        refused("sh_weight_grad_act8", *{**ok, **kw}.values(), match=match)

    bad("kept is NULL", kept=None)
    bad("dtype", dtype=0)
    bad("dtype", out_dtype=5)
    bad("dy is NULL", dy=0)
    bad("aligned", dy=P + 1)
    bad("dweight is NULL", dweight=0)
    bad("aligned", dweight=P + 2)
    bad("aligned", dbias=P + 2)
    bad("dw_ld", dw_ld=63)
    bad("out_features", out=1 << 22)
    bad("dy_ld", dy_ld=1 << 22)
    bad("workspace", ws=0)
    bad("workspace", ws_bytes=need.value - 1)
    bad("aligned", ws=P + 4)
    bad("too many", kept=kept(tokens=1 << 30))
    assert _native.lib().sh_weight_grad_act8(*{**ok, "out": 0, "dy": 0, "dweight": 0}.values()) == _native.SH_OK


def test_layer_norm_refusals():
    ok = dict.fromkeys(NORM_FIELDS, 0)
    for r in ("x", "y", "dy", "dx"):
        ok[f"{r}.data"] = P
    ok.update(stats=P, batch=2, seq=40, cols=64, dtype=1, weight_dtype=3, eps=1e-6)

    def pack(**kw):
        return layer_norm._ARGS.pack(*{**ok, **{k.replace("__", "."): v for k, v in kw.items()}}.values())

    def bad(match, which="both", **kw):
        if which != "backward":
            refused("sh_layer_norm", pack(**kw), 0, match=match)
        if which != "forward":
            refused("sh_layer_norm_backward", pack(**kw), P, 1 << 30, 0, match=match)

    refused("sh_layer_norm", None, 0, match="NULL")
    refused("sh_layer_norm_backward", None, P, 1 << 30, 0, match="NULL")
    refused("sh_layer_norm_workspace", None, ctypes.byref(ctypes.c_uint64()), match="NULL")
    refused("sh_layer_norm_workspace", pack(cols=16385), ctypes.byref(ctypes.c_uint64()), match="cols")
    refused("sh_layer_norm_workspace", pack(), None, match="NULL")
    bad("dtype", dtype=0)
    bad("weight_dtype", weight_dtype=9)
    bad("cols", cols=0)
    bad("cols", cols=16385)
    for eps in (-1e-9, float("inf"), float("nan")):
        bad("eps", eps=eps)
    bad("too many", batch=1 << 16, seq=1 << 16)
    bad("too many", batch=1 << 23, seq=1, per_batch=1)
    bad("aligned", weight=P + 2)
    bad("aligned", bias=P + 1)
    bad("aligned", "backward", dweight=P + 2)
    bad("aligned", "backward", dbias=P + 2)
    bad("aligned", stats=P + 2)
    bad("together", q=P)
    bad("together", exponent=P)
    bad("aligned", q=P + 8, exponent=P)
    bad("x is NULL", x__data=0)
    bad("aligned", x__data=P + 1)
    bad("y is NULL", "forward", y__data=0)
    bad("aligned", "forward", y__data=P + 1)
    bad("dy is NULL", "backward", dy__data=0)
    bad("aligned", "backward", dx__data=P + 1)
    bad("stats is NULL", "backward", stats=0)
    need = ctypes.c_uint64()
    args = pack(seq=4000, dweight=P)
    assert _native.lib().sh_layer_norm_workspace(args, ctypes.byref(need)) == _native.SH_OK and need.value > 0
    refused("sh_layer_norm_backward", args, P, need.value - 1, 0, match="workspace")
    refused("sh_layer_norm_backward", args, 0, need.value, 0, match="workspace")
    refused("sh_layer_norm_backward", args, P + 4, need.value, 0, match="aligned")
    assert _native.lib().sh_layer_norm_workspace(pack(seq=4000), ctypes.byref(need)) == _native.SH_OK and need.value == 0
    assert _native.lib().sh_layer_norm(pack(batch=0), 0) == _native.SH_OK
    assert _native.lib().sh_layer_norm_backward(pack(batch=0), 0, 0, 0) == _native.SH_OK


# ── streams ──────────────────────────────────────────────────────────────────


ON = torch.device("cuda", 1)
TENSOR = SimpleNamespace(is_cuda=True, device=ON)
KEPT = act8.Activation8(TENSOR, None, 1, torch.Size(()), torch.float32)


class Reached(Exception):
    pass


CALLS = [(act8, "quantize_activation", lambda f, s: f(TENSOR, stream=s)), (act8, "weight_grad_act8", lambda f, s: f(None, KEPT, stream=s)),
         (layer_norm, "layer_norm", lambda f, s: f(TENSOR, stream=s)), (act8.Activation8, "dequantize", lambda f, s: f(KEPT, stream=s))]


@pytest.mark.parametrize("owner,name,call", CALLS, ids=[c[1] for c in CALLS])
def test_a_stream_is_taken_on_the_tensors_device(monkeypatch, owner, name, call):
    made = []

    def stream(kind):
        def make(*args):
            made.append((kind, *args))
            return SimpleNamespace(device=args[-1])
        return make

    monkeypatch.setattr(torch.cuda, "ExternalStream", stream("external"))
    monkeypatch.setattr(torch.cuda, "default_stream", stream("default"))
    monkeypatch.setattr(torch.cuda, "stream", lambda s: made.append(("current", s.device)) or nullcontext())
    operator = getattr(owner, name)

    def inner(*args, **kw):  # the call on the current stream
        assert kw.get("stream") is None
        raise Reached

    monkeypatch.setattr(owner, name, inner)
    for given, want in ((77, [("external", 77, ON), ("current", ON)]), (0, [("default", ON), ("current", ON)]),
                        (SimpleNamespace(device=ON), [("current", ON)])):
        made.clear()
        with pytest.raises(Reached):
            call(operator, given)
        assert made == want
    made.clear()
    with pytest.raises(ValueError, match="cuda:0.*cuda:1"):
        call(operator, SimpleNamespace(device=torch.device("cuda", 0)))
    assert made == []


def test_host_tensors_are_refused():
    x = torch.zeros(4, 64)
    host = act8.Activation8(torch.zeros(4, 64, dtype=torch.int8), torch.ones(4, 2, dtype=torch.uint8), 64, torch.Size((4,)), torch.float32)
    for call in (lambda: act8.quantize_activation(x), lambda: layer_norm.layer_norm(x), lambda: host.dequantize(),
                 lambda: act8.weight_grad_act8(x, host), lambda: act8.linear_act8(x, x), lambda: act8.quantize_activation(x, stream=5),
                 lambda: layer_norm.layer_norm(x, stream=5), lambda: act8.checkpoint_act8(torch.sin, x.clone().requires_grad_())):
        with pytest.raises(ValueError, match="device"):
            call()


def test_gradients_whose_rows_overlap_are_refused():
    need = ctypes.c_uint64()
    assert _native.lib().sh_weight_grad_act8_workspace(kept(tokens=4096), 1, 33, 1, ctypes.byref(need)) == _native.SH_OK
    for ld in (0, 1, 32):
        refused("sh_weight_grad_act8", P, 1, ld, 33, kept(tokens=4096), P, 3, 64, P, P, need.value, 0, match="dy_ld")
