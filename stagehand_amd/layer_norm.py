"""Layer norm, plain, with weight and bias, or modulated by a scale and a shift for every sequence, with gradients.

For every token (the last dim of ``x``)::

    n = (x - mean(x)) / sqrt(var(x) + eps)
    y = n * weight + bias                   # n * (1 + weight) + bias when `modulate`

``var`` is the mean of the squared differences. Statistics, products and the gradients' sums are held in fp32; outputs
and gradients are rounded once. A mean far above the spread costs the output nothing; the backward pass takes the mean
rounded to fp32: there ``n`` is off by up to ``2**-24 * |mean| / sqrt(var + eps)``. The sum of a row and that of its squared
differences have to be numbers of fp32: values beyond 1e17, and where ``eps`` is 0 spreads below 1e-19, are outside it.

Everything runs on the caller's current torch stream unless ``stream`` is given. There is no CPU path.
"""
from __future__ import annotations

import ctypes
import struct

import torch
from torch.autograd.graph import increment_version

from stagehand_amd import _native
from stagehand_amd.act8 import GROUP
from stagehand_amd.int8 import DTYPE_CODES, check_no_grad, check_no_tangent, on_stream
from stagehand_amd.unpack import current_stream_handle

__all__ = ["layer_norm"]

MAX_COLS = 16384  # SH_LAYER_NORM_MAX_COLS
MAX_TOKENS = 0x7FFFFFFF

# Mirror of `struct sh_layer_norm_args`: four sh_rows, then pointers and strides, then 32-bit fields.
_ARGS = struct.Struct("<12Q" "7Q" "2Q" "7If")

_NO_ROWS = (0, 0, 0)


def _rows(t: torch.Tensor | None) -> tuple[int, int, int]:
    if t is None:
        return _NO_ROWS
    b, s, _ = t.stride()
    return t.data_ptr(), b, s


def _ptr(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


def _three_dims(t: torch.Tensor) -> torch.Tensor:
    """``t`` as (batch, seq, features) with contiguous rows; a copy only where strides ask for it."""
    if t.dim() != 3:
        t = t.reshape(1, t.numel() // t.shape[-1], t.shape[-1])
    return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


def _params(t: torch.Tensor | None, per_batch: bool) -> tuple[int, int, torch.Tensor | None]:
    """(address, elements between the sequences' rows, the tensor that holds them)."""
    if t is None:
        return 0, 0, None
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        t = t.contiguous()
    return t.data_ptr(), t.stride(0) if per_batch else 0, t


def _fields(shape, per_batch, modulate, eps, dtype, weight, bias) -> tuple:
    one = bias if weight is None else weight
    code = DTYPE_CODES[dtype]
    return (*shape, code, code if one is None else DTYPE_CODES[one.dtype], per_batch, modulate, eps)


def _forward(x, weight, bias, options, y, stats, q, exponent):
    per_batch, modulate, eps = options
    w, w_stride, weight = _params(weight, per_batch)
    b, b_stride, bias = _params(bias, per_batch)
    args = _ARGS.pack(*_rows(x), *_rows(y), *_NO_ROWS, *_NO_ROWS, w, b, 0, 0, _ptr(stats), _ptr(q), _ptr(exponent), w_stride, b_stride,
                      *_fields(x.shape, per_batch, modulate, eps, x.dtype, weight, bias))
    _native.check(_native.lib().sh_layer_norm(args, current_stream_handle()))


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, options, keep8):
        rows = _three_dims(x)
        batch, seq, cols = rows.shape
        y = x.new_empty(x.shape)
        stats = torch.empty((batch * seq, 2), dtype=torch.float32, device=x.device)
        q = exponent = None
        if keep8:
            groups = -(-cols // GROUP)
            q = torch.empty((batch * seq, groups * GROUP), dtype=torch.int8, device=x.device)
            exponent = torch.empty((batch * seq, groups), dtype=torch.uint8, device=x.device)
        _forward(rows, weight, bias, options, y.view(rows.shape), stats, q, exponent)
        ctx.save_for_backward(None if keep8 else x, weight, stats, q, exponent)
        ctx.options, ctx.dims, ctx.bias = options, (rows.shape, x.dtype), None if bias is None else (bias.shape, bias.dtype)
        return y

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():  # create_graph
            raise RuntimeError("layer_norm has no second derivatives")
        x, weight, stats, q, exponent = ctx.saved_tensors
        want_x, want_w, want_b = ctx.needs_input_grad[:3]
        shape, dtype = ctx.dims
        per_batch, modulate, eps = ctx.options
        dx = None
        if want_x:
            dx = torch.empty(dy.shape, dtype=dtype, device=dy.device)
        dw = torch.empty(weight.shape, dtype=weight.dtype, device=dy.device) if want_w else None
        db = torch.empty(ctx.bias[0], dtype=ctx.bias[1], device=dy.device) if want_b else None
        rows = None if x is None else _three_dims(x)
        dy = _three_dims(dy)
        w, w_stride, held = _params(weight, per_batch)
        code = DTYPE_CODES[dtype]
        params = code if weight is None and ctx.bias is None else DTYPE_CODES[ctx.bias[1] if weight is None else weight.dtype]
        args = _ARGS.pack(*_rows(rows), *_NO_ROWS, *_rows(dy), *_rows(None if dx is None else dx.view(shape)), w, 0, _ptr(dw), _ptr(db),
                          stats.data_ptr(), _ptr(q), _ptr(exponent), w_stride, 0, *shape, code, params, per_batch, modulate, eps)
        lib, need, ws = _native.lib(), ctypes.c_uint64(), None
        if want_w or want_b:
            _native.check(lib.sh_layer_norm_workspace(args, ctypes.byref(need)))
            if need.value:
                ws = torch.empty(need.value, dtype=torch.uint8, device=dy.device)
        _native.check(lib.sh_layer_norm_backward(args, _ptr(ws), need.value, current_stream_handle()))
        return dx, dw, db, None, None


def _check_params(t: torch.Tensor, what: str, device: int, shape: torch.Size) -> bool:
    """Whether ``t`` has a row for every sequence."""
    cols = shape[-1]
    if t.get_device() != device or t.dtype not in DTYPE_CODES:
        raise ValueError(f"{what} must be bfloat16, float16 or float32 on x's device, got {t.device} {t.dtype}")
    if t.dim() and t.shape[-1] == cols and t.numel() == cols:
        return False
    if len(shape) == 3 and tuple(t.shape) in ((shape[0], cols), (shape[0], 1, cols)):
        return True
    rows = f", ({shape[0]}, {cols}) or ({shape[0]}, 1, {cols})" if len(shape) == 3 else ""
    raise ValueError(f"{what} must be ({cols},){rows} for x {tuple(shape)}, got {tuple(t.shape)}")


def _overlap(t: torch.Tensor) -> bool:
    """Whether rows of ``t`` (batch, seq, features) may share memory."""
    if t.numel() == 0:
        return False
    reach = t.shape[2]
    for stride, size in sorted(zip(t.stride()[:2], t.shape)):
        if size > 1:
            if stride < reach:
                return True
            reach += (size - 1) * stride
    return False


def layer_norm(
    x: torch.Tensor,
    weight: torch.Tensor | None = None,
    bias: torch.Tensor | None = None,
    *,
    eps: float = 1e-6,
    modulate: bool = False,
    keep8: bool = False,
    out: torch.Tensor | None = None,
    stream: torch.cuda.Stream | int | None = None,
) -> torch.Tensor:
    """The layer norm of ``x`` over its last dim; see the module's formulas.

    ``weight`` and ``bias`` (of one type, each optional) hold a value for every feature or, for ``x`` of three dims
    ``(batch, seq, features)``, a row ``(batch, features)`` or ``(batch, 1, features)`` for every sequence: what a block's
    modulation gives, as the chunks that it is split into. With ``modulate`` the gain is ``1 + weight``.

    ``keep8`` keeps ``x`` in 8 bits for the backward pass instead of the tensor itself, as
    :func:`stagehand_amd.act8.quantize_activation` does, written in the forward's pass over ``x``: the output is the same,
    the gradients are those at the kept values, with the mean and variance of ``x``.

    Rows of a larger tensor are read in place. The output is contiguous, or written to ``out``: a tensor of the same shape
    and type whose rows are contiguous (``x`` itself, but no other memory of the inputs'). A backward pass that needs
    the old values of ``out`` raises. Gradients flow to ``x``, ``weight`` and ``bias``, not through ``out``."""
    if stream is not None:
        with on_stream(stream, x):
            return layer_norm(x, weight, bias, eps=eps, modulate=modulate, keep8=keep8, out=out)
    device, shape, dtype = x.get_device(), x.shape, x.dtype
    if device < 0 or not shape or dtype not in DTYPE_CODES:
        raise ValueError(f"x must be a device tensor (..., features) in bfloat16, float16 or float32, got {x.device} {dtype} {tuple(shape)}")
    cols = shape[-1]
    if not 1 <= cols <= MAX_COLS:
        raise ValueError(f"features {cols} are not in 1 .. {MAX_COLS}")
    tokens = x.numel() // cols
    if tokens > MAX_TOKENS:
        raise ValueError(f"x must have at most {MAX_TOKENS} tokens, got {tokens}")
    per_batch = False
    if weight is not None:
        per_batch = _check_params(weight, "weight", device, shape)
    if bias is not None:
        rows = _check_params(bias, "bias", device, shape)
        if weight is not None and (rows != per_batch or bias.dtype != weight.dtype):
            raise ValueError(f"weight and bias must have one type, and both a row for every sequence or neither, got {weight.dtype} "
                             f"{tuple(weight.shape)} and {bias.dtype} {tuple(bias.shape)}")
        per_batch = rows
    if not 0.0 <= eps <= 1e38:
        raise ValueError(f"eps {eps} is negative or not finite")
    check_no_tangent("layer_norm", x, weight, bias)
    if device != torch.cuda.current_device():
        with torch.cuda.device(device):
            return layer_norm(x, weight, bias, eps=eps, modulate=modulate, keep8=keep8, out=out)
    options = per_batch, bool(modulate), eps
    grad = torch.is_grad_enabled() and any([t is not None and t.requires_grad for t in (x, weight, bias)])
    if out is None:
        if grad:
            return _LayerNorm.apply(x, weight, bias, options, bool(keep8))
        y = x.new_empty(shape)
        rows, y_rows = _three_dims(x), y.view(1, tokens, cols) if len(shape) != 3 else y
    else:
        if grad:
            raise RuntimeError("out= has no gradient: call layer_norm under torch.no_grad(), or without out")
        if out.get_device() != device or out.shape != shape or out.dtype != dtype:
            raise ValueError(f"out must be {dtype} {tuple(shape)} on x's device, got {out.device} {out.dtype} {tuple(out.shape)}")
        check_no_grad(out, "out")
        check_no_tangent("out", out)
        try:
            y_rows = out if len(shape) == 3 else out.view(1, tokens, cols)
        except RuntimeError:
            y_rows = None
        if y_rows is None or (cols > 1 and y_rows.stride(2) != 1) or _overlap(y_rows):
            raise ValueError(f"out must be rows of contiguous values that share no memory, got strides {out.stride()}")
        rows, y = _three_dims(x), out
    _forward(rows, weight, bias, options, y_rows, None, None, None)
    if out is not None:
        increment_version(out)
    return y
