"""Activations kept in 8 bits for the backward pass, and what reads them there.

Training keeps activations from the forward for the backward pass. Here they are kept in 8.25 bits a value
instead of 16 or 32: groups of 32 neighbouring features share a power of two ``2**k``, the smallest with ``max |x| <=
127 * 2**k`` (``k`` from -126 on), and are rounded to whole multiples of it, ties to even::

    kept = quantize_activation(x)                   # an Activation8
    x_again = kept.dequantize()                     # off by at most half of the group's 2**k

The rounding to a multiple is the only one: what is kept of a bfloat16, float16 or float32 tensor is a tensor of that
type. (Where ``64 * 2**k`` is no number of the type any more, for values near its largest, multiples end
with 63.) A group with an infinity or a NaN is read back as NaNs.

Three things read kept activations in the backward pass:

- :func:`checkpoint_act8` recomputes a function from its kept input, as activation checkpointing does;
- :func:`linear_act8`, a Linear layer that keeps its input in 8 bits: the gradient of its weight is multiplied from
  what is kept as it is (:func:`weight_grad_act8`), on the matrix cores;
- :func:`stagehand_amd.layer_norm.layer_norm` with ``keep8``.

Everything runs on the caller's current torch stream unless ``stream`` is given; outputs and workspaces are
allocated on that stream. There is no CPU path.
"""
from __future__ import annotations

import ctypes
import math
import struct
from typing import Any, Callable, NamedTuple

import torch
from torch.autograd.graph import increment_version
from torch.nn import functional as F

from stagehand_amd import _native
from stagehand_amd.int8 import DTYPE_CODES, _output, _token_rows, check_device, check_no_tangent, on_stream
from stagehand_amd.unpack import current_stream_handle

__all__ = ["Activation8", "quantize_activation", "weight_grad_act8", "linear_act8", "checkpoint_act8"]

GROUP = 32  # SH_ACT8_GROUP
MAX_COLS = 0x00FFFFFF  # SH_ACT8_MAX_COLS
MAX_OUT = 0x003FFFFF  # SH_WEIGHT_GRAD_MAX_OUT

_KEPT = struct.Struct("<2Q2I")  # mirror of `struct sh_act8`


class Activation8(NamedTuple):
    """An activation kept in 8 bits: the value of feature ``i`` of a token is ``q[i] * 2**(exponent[i // 32] - 127)``."""

    q: torch.Tensor         # int8 (tokens, features rounded up to 32), zeros past the features
    exponent: torch.Tensor  # uint8 (tokens, groups): k + 127; 255: the group is NaN
    features: int
    shape: torch.Size       # of the activation, without the last dim
    dtype: torch.dtype      # of the activation

    @property
    def nbytes(self) -> int:
        return self.q.numel() + self.exponent.numel()

    def dequantize(self, dtype: torch.dtype | None = None, out: torch.Tensor | None = None,
                   stream: torch.cuda.Stream | int | None = None) -> torch.Tensor:
        """The kept values in ``dtype`` (default: the activation's, in which they are exact, or that of ``out``)."""
        if stream is not None:
            with on_stream(stream, self.q):
                return self.dequantize(dtype, out)
        if dtype is None:
            dtype = self.dtype if out is None else out.dtype
        if dtype not in DTYPE_CODES:
            raise ValueError(f"dtype must be bfloat16, float16 or float32, got {dtype}")
        args, index = _kept_args(self)
        if index != torch.cuda.current_device():
            with torch.cuda.device(index):
                return self.dequantize(dtype, out)
        if out is None:
            y, ld = self.q.new_empty((*self.shape, self.features), dtype=dtype), self.features
        else:
            y, ld = _output(out, (*self.shape, self.features), dtype, self.q.device)
        _native.check(_native.lib().sh_act8_dequantize(args, y.data_ptr(), DTYPE_CODES[dtype], ld, current_stream_handle()))
        if out is not None:
            increment_version(out)
        return y


def _kept_args(kept: Activation8) -> tuple[bytes, int]:
    """(``struct sh_act8``, the device's index), after a look at what the tuple holds."""
    q, exponent, features, shape, dtype = kept
    if not 1 <= features <= MAX_COLS:
        raise ValueError(f"a token must have 1 .. {MAX_COLS} features, got {features}")
    groups, tokens = -(-features // GROUP), math.prod(shape)
    index = q.get_device()
    if index < 0 or exponent.get_device() != index:
        raise ValueError(f"kept.q and kept.exponent must be on one device, got {q.device} and {exponent.device}")
    if q.dtype != torch.int8 or exponent.dtype != torch.uint8 or q.shape != (tokens, groups * GROUP) or \
            exponent.shape != (tokens, groups) or not q.is_contiguous() or not exponent.is_contiguous():
        raise ValueError(f"kept must hold contiguous int8 {(tokens, groups * GROUP)} and uint8 {(tokens, groups)}, got {q.dtype} "
                         f"{tuple(q.shape)} and {exponent.dtype} {tuple(exponent.shape)}")
    if dtype not in DTYPE_CODES:
        raise ValueError(f"kept.dtype must be bfloat16, float16 or float32, got {dtype}")
    return _KEPT.pack(q.data_ptr(), exponent.data_ptr(), tokens, features), index


def quantize_activation(x: torch.Tensor, stream: torch.cuda.Stream | int | None = None) -> Activation8:
    """Keeps ``x`` (any leading dims, features last) in 8 bits; see the module's text.

    The result has no gradient: a call that would have to record one is refused."""
    if stream is not None:
        with on_stream(stream, x):
            return quantize_activation(x)
    code = DTYPE_CODES.get(x.dtype)
    if code is None:
        raise ValueError(f"x must be bfloat16, float16 or float32, got {x.dtype}")
    if x.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("quantize_activation has no gradient: call it under torch.no_grad(), or on x.detach()")
    check_no_tangent("quantize_activation", x)
    index, shape = x.get_device(), x.shape
    if index < 0:
        raise ValueError(f"x must be a device tensor, got {x.device}")
    rows, tokens, ld = _token_rows(x, "x")
    features = rows.shape[1]
    if not 1 <= features <= MAX_COLS:
        raise ValueError(f"a token must have 1 .. {MAX_COLS} features, got {features}")
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            return quantize_activation(x)
    groups = -(-features // GROUP)
    q = x.new_empty((tokens, groups * GROUP), dtype=torch.int8)
    exponent = x.new_empty((tokens, groups), dtype=torch.uint8)
    kept = _KEPT.pack(q.data_ptr(), exponent.data_ptr(), tokens, features)
    _native.check(_native.lib().sh_act8_quantize(rows.data_ptr(), code, ld, kept, current_stream_handle()))
    return Activation8(q, exponent, features, shape[:-1], x.dtype)


def weight_grad_act8(dy: torch.Tensor, kept: Activation8, *, bias: bool = False, out_dtype: torch.dtype | None = None,
                     stream: torch.cuda.Stream | int | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """The gradients ``(dweight, dbias)`` of a Linear from the gradient ``dy`` of its output and its kept input:
    ``dweight[o, i] = sum dy[..., o] * kept[..., i]``, ``dbias[o] = sum dy[..., o]`` (None without ``bias``).

    ``dy`` has the kept activation's type and leading dims. The products are summed in float32 in a fixed order and
    rounded once to ``out_dtype`` (default: the type of ``dy``). A float32 ``dy`` is multiplied with all its bits from ``2**-110``
    on; of smaller values, what lies under ``2**-133`` is cut in ``dweight``."""
    if stream is not None:
        with on_stream(stream, kept.q):
            return weight_grad_act8(dy, kept, bias=bias, out_dtype=out_dtype)
    args, index = _kept_args(kept)
    if dy.dtype != kept.dtype:
        raise ValueError(f"dy must have the kept activation's type {kept.dtype}, got {dy.dtype}")
    if dy.dim() == 0 or dy.shape[:-1] != kept.shape:
        raise ValueError(f"dy must have the kept activation's leading dims {tuple(kept.shape)}, got {tuple(dy.shape)}")
    if out_dtype is None:
        out_dtype = dy.dtype
    elif out_dtype not in DTYPE_CODES:
        raise ValueError(f"out_dtype must be bfloat16, float16 or float32, got {out_dtype}")
    if dy.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("weight_grad_act8 has no gradient: call it under torch.no_grad(), or on dy.detach()")
    check_no_tangent("weight_grad_act8", dy)
    if dy.get_device() != index:
        raise ValueError(f"dy must be on {kept.q.device}, got {dy.device}")
    out, features = dy.shape[-1], kept.features
    if out > MAX_OUT:
        raise ValueError(f"dy must have at most {MAX_OUT} features, got {out}")
    rows, tokens, ld = _token_rows(dy, "dy")
    if tokens > 1 and not out <= ld <= MAX_OUT:  # rows that share memory, as of a sum's gradient, or lie too far apart
        rows, ld = rows.contiguous(), out
    elif tokens <= 1:
        ld = out
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            return weight_grad_act8(dy, kept, bias=bias, out_dtype=out_dtype)
    code = DTYPE_CODES[dy.dtype]
    dw = dy.new_empty((out, features), dtype=out_dtype)
    db = dy.new_empty(out, dtype=out_dtype) if bias else None
    lib, need = _native.lib(), ctypes.c_uint64()
    _native.check(lib.sh_weight_grad_act8_workspace(args, code, out, bool(bias), ctypes.byref(need)))
    ws = dy.new_empty(need.value, dtype=torch.uint8) if need.value else None
    _native.check(lib.sh_weight_grad_act8(rows.data_ptr(), code, ld, out, args, dw.data_ptr(), DTYPE_CODES[out_dtype], features,
                                          None if db is None else db.data_ptr(), None if ws is None else ws.data_ptr(),
                                          need.value, current_stream_handle()))
    return dw, db


def _bias_grad(dy: torch.Tensor) -> torch.Tensor:
    """The sum of ``dy`` over its tokens.

    torch's sum over many blocks clears its flags with a memset, which a captured graph does not repeat rightly: its replays
    after the first are wrong. Into a graph go the weight gradient's kernels, with one input feature of no meaning, whose
    gradient is dropped (16384 tokens x 4096 in bf16 38 us, torch's 37; x 64 71 us, torch's 11)."""
    shape = dy.shape[:-1]
    tokens = math.prod(shape)
    if not torch.cuda.is_current_stream_capturing():
        return dy.reshape(tokens, dy.shape[-1]).sum(0)
    q, exponent = dy.new_empty((tokens, GROUP), dtype=torch.int8), dy.new_empty((tokens, 1), dtype=torch.uint8)
    return weight_grad_act8(dy, Activation8(q, exponent, 1, shape, dy.dtype), bias=True)[1]


class _LinearAct8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, kept):
        want_x, want_weight, want_bias = ctx.needs_input_grad[:3]
        if want_weight and kept is None:
            kept = quantize_activation(x)
        q, exponent = kept[:2] if want_weight else (None, None)
        ctx.rest = kept[2:] if want_weight else None
        ctx.save_for_backward(weight if want_x else None, q, exponent)
        return F.linear(x, weight, bias)

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():  # create_graph
            raise RuntimeError("linear_act8 has no second derivatives")
        weight, q, exponent = ctx.saved_tensors
        want_x, want_weight, want_bias = ctx.needs_input_grad[:3]
        dx = dw = db = None
        if want_x:  # in two dims: a plain product, whatever dy's strides
            tokens = math.prod(dy.shape[:-1])
            dx = (dy.reshape(tokens, dy.shape[-1]) @ weight).view(*dy.shape[:-1], weight.shape[1])
        if want_weight:
            dw, db = weight_grad_act8(dy, Activation8(q, exponent, *ctx.rest), bias=want_bias)
        elif want_bias:
            db = _bias_grad(dy)
        return dx, dw, db, None


def linear_act8(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
                kept: Activation8 | None = None) -> torch.Tensor:
    """``torch.nn.functional.linear(x, weight, bias)`` that keeps its input in 8 bits for the weight's gradient.

    The output and the gradients of ``x`` and ``bias`` are those of an ordinary Linear, the gradient of ``weight`` that of one
    whose input were ``kept.dequantize()``. Layers with one input share what is kept of it: ``kept`` is
    ``quantize_activation(x.detach())``, made once. Nothing is kept when ``weight`` needs no gradient, or without grad mode.
    Under autocast, inputs are cast as for an ordinary Linear (``kept`` then holds the cast input)."""
    if torch.is_autocast_enabled("cuda"):
        dtype = torch.get_autocast_dtype("cuda")
        for what, t in (("x", x), ("weight", weight), ("bias", bias)):
            if t is not None and t.dtype not in DTYPE_CODES:  # autocast leaves these as they are
                raise ValueError(f"{what} must be of type bfloat16, float16 or float32, got {t.dtype}")
        with torch.autocast("cuda", enabled=False):
            return linear_act8(x.to(dtype), weight.to(dtype), None if bias is None else bias.to(dtype), kept)
    check_device(x, None, "x")
    if x.dtype not in DTYPE_CODES or weight.dtype != x.dtype or (bias is not None and bias.dtype != x.dtype):
        raise ValueError(f"x, weight and bias must have one type of bfloat16, float16 and float32, got {x.dtype}, {weight.dtype}"
                         f"{'' if bias is None else f' and {bias.dtype}'}")
    if x.dim() == 0 or weight.dim() != 2 or weight.shape[1] != x.shape[-1] or (bias is not None and bias.shape != weight.shape[:1]):
        raise ValueError(f"weight must be (out, {x.shape[-1] if x.dim() else '?'}) and bias (out,), got {tuple(weight.shape)}"
                         f"{'' if bias is None else f' and {tuple(bias.shape)}'}")
    check_device(weight, x.device, "weight")
    if bias is not None:
        check_device(bias, x.device, "bias")
    check_no_tangent("linear_act8", x, weight, bias)
    if kept is not None:
        if kept.dtype != x.dtype or kept.features != x.shape[-1] or torch.Size(kept.shape) != x.shape[:-1]:
            raise ValueError(f"kept is of a {kept.dtype} {(*kept.shape, kept.features)} activation, x is {x.dtype} {tuple(x.shape)}")
        check_device(kept.q, x.device, "kept.q")
    if not torch.is_grad_enabled():  # a Function's needs_input_grad does not look at this
        return F.linear(x, weight, bias)
    return _LinearAct8.apply(x, weight, bias, kept)


def checkpoint_act8(function: Callable[..., Any], x: torch.Tensor, *args: Any, **kwargs: Any) -> Any:
    """``function(x, *args, **kwargs)``, of which only ``x`` is kept for the backward pass, in 8 bits: the backward pass
    recomputes the rest from ``quantize_activation(x).dequantize()``, whose dims lie in memory in the order of those of ``x``.

    As ``torch.utils.checkpoint.checkpoint`` without reentrance, to which it leaves the recomputation (random state and
    autocast are restored); ``args`` and ``kwargs`` are kept as they are. ``function`` must not write to ``x``. The
    output is that of ``function`` itself; gradients are those at the kept input."""
    if not torch.is_grad_enabled():
        return function(x, *args, **kwargs)
    from torch.utils.checkpoint import checkpoint

    check_no_tangent("checkpoint_act8", x)
    kept = quantize_activation(x.detach())
    needs_grad, first = x.requires_grad, [x]
    strides = None if x.is_contiguous() else torch.empty_like(x, device="meta").stride()  # dense, dims in the order of x's

    def run(q: torch.Tensor, *rest: Any) -> Any:
        # the forward pass runs on x itself, a recomputation on what is kept of it
        if first:
            return function(first[0], *rest, **kwargs)
        again = kept.dequantize()
        if strides is not None and again.stride() != strides:  # views that x's order of dims allows stay views
            again = torch.empty_strided(again.shape, strides, dtype=again.dtype, device=again.device).copy_(again)
        return function(again.requires_grad_(needs_grad), *rest, **kwargs)

    try:
        return checkpoint(run, kept.q, *args, use_reentrant=False)  # q tells it the device
    finally:
        first.clear()
