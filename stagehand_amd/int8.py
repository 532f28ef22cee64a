"""Linear layers on SquareQ weights that stay in int8 on the device.

A SquareQ row is int8 values with one fp32 scale and, at times, a zero point: ``W[n][k] =
(q[n][k] - zero_point[n]) * scale[n]`` (src/stagehand/scheduler.py:285-308). :mod:`stagehand_amd.unpack`
turns such rows into bf16; here they are multiplied as they are. The activations are quantised to
int8 too, one scale per token, the products are summed exactly in 32-bit integers, and scales, zero
points and bias are applied once at the end in fp32::

    weight = Int8Weight(qweight, scale, zero_point=zp, bias=bias)   # kept for the layer's life
    y = linear_i8(x, weight)                                        # any leading dims, y in x's type

``quantize_tokens`` and ``matmul_i8`` are its two halves, for activations that go into several
products. The product is for inference: the rounding to int8 has no gradient, so a call that would
have to record one is refused.

Everything runs on the caller's current torch stream unless ``stream`` is given; outputs and
workspaces are allocated on that stream. As with any torch operator, inputs that were made on
another stream must be ready, and kept, for it. ``out`` is written in place: it must not share memory
with the inputs, and a backward pass that needs its old values raises. There is no CPU path.
"""
from __future__ import annotations

import ctypes
from typing import Any, NamedTuple

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from stagehand_amd import _native
from stagehand_amd.unpack import current_stream_handle

__all__ = ["Int8Weight", "Int8Tokens", "quantize_tokens", "matmul_i8", "linear_i8"]

MAX_COLS = 131071  # SH_I8_MAX_COLS
TOKEN_ALIGN = 128  # SH_I8_TOKEN_ALIGN
MAX_LD = 1 << 20  # bytes between rows
INTEGERS = (torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64)
DTYPE_CODES = {torch.bfloat16: 1, torch.float16: 2, torch.float32: 3}  # enum sh_dtype


class _Weight(ctypes.Structure):
    """Mirror of ``struct sh_i8_weight``."""

    _fields_ = [("q", ctypes.c_void_p), ("ld", ctypes.c_uint64), ("rows", ctypes.c_uint32), ("cols", ctypes.c_uint32),
                ("scale", ctypes.c_void_p), ("zero_point", ctypes.c_void_p), ("bias", ctypes.c_void_p)]


def on_stream(stream: torch.cuda.Stream | int, t: torch.Tensor):
    """Context in which ``stream`` (a torch stream, or a raw handle on the device of ``t``) is torch's current
    stream, for a call that works on ``t``."""
    check_device(t, None, "a tensor for the stream")
    if isinstance(stream, int):  # ExternalStream(0) would be a new stream
        stream = torch.cuda.ExternalStream(stream, t.device) if stream else torch.cuda.default_stream(t.device)
    elif stream.device != t.device:
        raise ValueError(f"the stream is on {stream.device}, the tensors on {t.device}")
    return torch.cuda.stream(stream)


def check_device(t: torch.Tensor, device: torch.device | None, what: str) -> None:
    if not t.is_cuda:
        raise ValueError(f"{what} must be a device tensor, got {t.device}")
    if device is not None and t.device != device:
        raise ValueError(f"{what} is on {t.device}, not on {device}")


def check_no_tangent(who: str, *tensors: torch.Tensor | None) -> None:
    """Refuses dual tensors: their ``requires_grad`` is False, and a result without a tangent says that the derivative is 0."""
    if getattr(forward_ad, "_current_level", 0) < 0:  # no dual tensors exist; 0.03 us instead of 0.3 a tensor
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{who} has no forward-mode derivatives")


def check_no_grad(t: torch.Tensor, what: str) -> None:
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{what} requires grad, but what is written to it has no gradient: call under torch.no_grad()")


class Int8Weight:
    """A SquareQ weight in device memory, as :func:`linear_i8` takes it.

    ``qweight`` is int8 ``(out_features, padded_in)``; ``in_features`` of its columns count (default:
    all). ``scale`` and the optional ``zero_point`` and ``bias`` hold ``out_features`` values; they are
    constants here (no gradient), kept in fp32; zero points may be integers. ``qweight`` is used where it
    lies if its rows start on 128-byte boundaries and its memory holds all of the last row; changes of it
    are then seen by later calls. Otherwise it is copied once into such rows. With ``realign=False`` rows
    that start on 16-byte boundaries are used where they lie too: no copy, and 7% slower products of many
    tokens (4608 x 21504 x 3072: 288 us against 268), for a weight that is multiplied a few times only.
    """

    def __init__(self, qweight: torch.Tensor, scale: torch.Tensor, zero_point: torch.Tensor | None = None,
                 bias: torch.Tensor | None = None, in_features: int | None = None, realign: bool = True) -> None:
        if qweight.dtype != torch.int8 or qweight.dim() != 2:
            raise ValueError(f"qweight must be a 2-D int8 tensor, got {qweight.dim()}-D {qweight.dtype}")
        check_device(qweight, None, "qweight")
        rows, width = qweight.shape
        _count(rows, "qweight's rows")
        cols = width if in_features is None else int(in_features)
        if not 1 <= cols <= min(width, MAX_COLS):
            raise ValueError(f"in_features {cols} is not in 1 .. {min(width, MAX_COLS)}")
        self.out_features, self.in_features, self.device = rows, cols, qweight.device
        align = 128 if realign else 16
        self.qweight = _aligned_rows(qweight[:, :cols], align)
        self.scale = self._per_row(scale, "scale")
        if zero_point is not None and zero_point.dtype in INTEGERS:
            zero_point = zero_point.float()
        self.zero_point = None if zero_point is None else self._per_row(zero_point, "zero_point")
        self.bias = None if bias is None else self._per_row(bias, "bias")
        ld = self.qweight.stride(0) if rows > 1 else _round_up(cols, align)
        self._struct = _Weight(self.qweight.data_ptr(), ld, rows, cols, self.scale.data_ptr(),
                               0 if self.zero_point is None else self.zero_point.data_ptr(),
                               0 if self.bias is None else self.bias.data_ptr())
        self._ref = ctypes.addressof(self._struct)

    def _per_row(self, t: torch.Tensor, what: str) -> torch.Tensor:
        if t.numel() != self.out_features:
            raise ValueError(f"{what} must hold {self.out_features} values, got {t.numel()}")
        if not t.dtype.is_floating_point:
            raise ValueError(f"{what} must be floating point, got {t.dtype}")
        return t.detach().to(device=self.device, dtype=torch.float32).reshape(-1).contiguous()

    @classmethod
    def from_squareq(cls, layer: dict[str, Any], out_features: int | None = None, in_features: int | None = None,
                     device: torch.device | str = "cuda", realign: bool = True) -> "Int8Weight":
        """A layer of a SquareQ slab ({"qweight", "scale", ["zero_point"], ["bias"]}, the layer dict of
        src/stagehand/scheduler.py:285-308 and of :func:`stagehand_amd.squareq_v2.read_v2_layers`) on
        ``device``. Rows past ``out_features`` and columns past ``in_features`` are padding. Zero points
        that are all 0 are dropped."""
        q = layer["qweight"]
        q = q.reshape(q.shape[0], -1)
        rows = q.shape[0] if out_features is None else int(out_features)
        if not 0 <= rows <= q.shape[0]:
            raise ValueError(f"out_features {rows} is not in 0 .. {q.shape[0]}")
        zp, bias = layer.get("zero_point"), layer.get("bias")
        if zp is not None:
            zp = zp.reshape(-1)[:rows]
            if not bool((zp != 0).any()):
                zp = None
        return cls(q[:rows].to(device), layer["scale"].reshape(-1)[:rows], None if zp is None else zp,
                   None if bias is None else bias.reshape(-1)[:rows], in_features, realign)

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """``(q - zero_point) * scale``, computed in fp32 and rounded to ``dtype``."""
        w = self.qweight.float()
        if self.zero_point is not None:
            w -= self.zero_point[:, None]
        return (w * self.scale[:, None]).to(dtype)


def _count(n: int, what: str) -> int:
    """``n`` as the C calls take it, in 32 bits (ctypes would pass on its lower half)."""
    if n > 0xFFFFFFFF:
        raise ValueError(f"{what} must be at most {0xFFFFFFFF}, got {n}")
    return n


def _round_up(n: int, m: int) -> int:
    return -(-n // m) * m


def _aligned_rows(q: torch.Tensor, align: int) -> torch.Tensor:
    """``q`` itself where its rows start on multiples of ``align`` bytes, else a copy in such rows."""
    rows, cols = q.shape
    ld = q.stride(0) if rows > 1 else _round_up(cols, align)
    if (cols == 1 or q.stride(1) == 1) and ld % align == 0 and cols <= ld <= MAX_LD and q.data_ptr() % align == 0 and \
            q.untyped_storage().nbytes() - q.storage_offset() >= rows * ld:
        return q
    padded = torch.zeros((rows, _round_up(cols, align)), dtype=torch.int8, device=q.device)
    padded[:, :cols] = q
    return padded[:, :cols]


class Int8Tokens(NamedTuple):
    """Quantised activations: ``x ≈ q[:, :in_features] * scale[:, None]``."""

    q: torch.Tensor      # int8 (tokens, in_features rounded up to 128), zeros past in_features
    scale: torch.Tensor  # float32 (tokens,)
    sums: torch.Tensor   # int32 (tokens,): sum of each token's q
    in_features: int
    shape: torch.Size    # of the activations, without the last dim

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        x = self.q[:, :self.in_features] * self.scale[:, None]
        return x.to(dtype).reshape(*self.shape, self.in_features)


def _token_rows(x: torch.Tensor, what: str) -> tuple[torch.Tensor, int, int]:
    """(x as rows of contiguous values, tokens, elements between rows); a copy only where strides ask for it."""
    if x.dim() == 0:
        raise ValueError(f"{what} must have at least one dimension")
    if x.dim() != 2:
        x = x.reshape(x.numel() // x.shape[-1] if x.shape[-1] else 0, x.shape[-1])
    if x.shape[1] > 1 and x.stride(1) != 1:
        x = x.contiguous()
    return x, _count(x.shape[0], f"{what}'s tokens"), x.stride(0)


def _check_input(x: torch.Tensor, who: str) -> int:
    code = DTYPE_CODES.get(x.dtype)
    if code is None:
        raise ValueError(f"x must be bfloat16, float16 or float32, got {x.dtype}")
    if x.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{who} is for inference and has no gradient: call it under torch.no_grad(), or on x.detach()")
    check_no_tangent(who, x)
    return code


def _output(out: torch.Tensor | None, shape: tuple[int, ...], dtype: torch.dtype,
            device: torch.device) -> tuple[torch.Tensor, int]:
    """(the output, elements between its rows)."""
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=device)
        return out, shape[-1]
    check_device(out, device, "out")
    check_no_grad(out, "out")
    check_no_tangent("out", out)
    if tuple(out.shape) != tuple(shape) or out.dtype != dtype:
        raise ValueError(f"out must be {dtype} {tuple(shape)}, got {out.dtype} {tuple(out.shape)}")
    try:
        rows = out.view(-1, shape[-1]) if out.numel() else out.reshape(0, shape[-1])
    except RuntimeError:
        rows = None
    if rows is None or (shape[-1] > 1 and rows.numel() and rows.stride(1) != 1):
        raise ValueError(f"out must be rows of contiguous values at one distance, got strides {out.stride()}")
    return out, rows.stride(0) if rows.shape[0] > 1 else shape[-1]


def quantize_tokens(x: torch.Tensor, stream: torch.cuda.Stream | int | None = None) -> Int8Tokens:
    """Quantises every token (the last dim of ``x``) to int8 with one scale: ``a = max |x|``, ``q =
    rint(x * (127 / a))``, ``scale = a / 127``.

    A token with ``a < 2**-120`` counts as zero (q and scale 0). A token with an infinity or a NaN gets
    q = 0 and scale NaN, so every product of it is NaN."""
    if stream is not None:
        with on_stream(stream, x):
            return quantize_tokens(x)
    code = _check_input(x, "quantize_tokens")
    check_device(x, None, "x")
    rows, tokens, ld = _token_rows(x, "x")
    cols = rows.shape[1]
    if not 1 <= cols <= MAX_COLS:
        raise ValueError(f"a token must have 1 .. {MAX_COLS} values, got {cols}")
    q_ld = _round_up(cols, TOKEN_ALIGN)
    with torch.cuda.device(x.device):
        q = torch.empty((tokens, q_ld), dtype=torch.int8, device=x.device)
        scale = torch.empty(tokens, dtype=torch.float32, device=x.device)
        sums = torch.empty(tokens, dtype=torch.int32, device=x.device)
        _native.call("sh_quantize_tokens", rows.data_ptr(), code, ld, tokens, cols, q.data_ptr(), q_ld,
                     scale.data_ptr(), sums.data_ptr(), current_stream_handle())
    return Int8Tokens(q, scale, sums, cols, x.shape[:-1])


def matmul_i8(tokens: Int8Tokens, weight: Int8Weight, out: torch.Tensor | None = None,
              out_dtype: torch.dtype | None = None, stream: torch.cuda.Stream | int | None = None) -> torch.Tensor:
    """``tokens · weightᵀ + bias`` in ``out_dtype`` (default bfloat16, or that of ``out``).

    ``tokens.q`` may be rows of a larger tensor (every second token, the last one of each sequence, some of
    its columns): rows on multiples of 128 bytes, up to 1 MiB apart, are read in place, others are copied."""
    if stream is not None:
        with on_stream(stream, weight.qweight):
            return matmul_i8(tokens, weight, out, out_dtype)
    q, scale, sums, cols, shape = tokens
    if cols != weight.in_features:
        raise ValueError(f"the tokens have {cols} values, the weight takes {weight.in_features}")
    n = _count(q.shape[0], "the tokens of tokens.q") if q.dim() == 2 else -1
    width = _round_up(cols, TOKEN_ALIGN)
    if q.dtype != torch.int8 or n < 0 or q.shape[1] < width or (q.numel() and q.stride(1) != 1):
        raise ValueError(f"tokens.q must be int8 rows of {cols} values and zeros up to {width}, got {q.dtype} {tuple(q.shape)}")
    if scale.dtype != torch.float32 or sums.dtype != torch.int32 or scale.shape != (n,) or sums.shape != (n,) or \
            not scale.is_contiguous() or not sums.is_contiguous():
        raise ValueError("tokens.scale and tokens.sums must be contiguous float32 and int32 with one value per token")
    if scale.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("matmul_i8 is for inference and has no gradient: call it under torch.no_grad()")
    check_no_tangent("matmul_i8", scale)
    if torch.Size(shape).numel() != n:
        raise ValueError(f"tokens.shape {tuple(shape)} does not hold {n} tokens")
    for what, t in (("tokens.q", q), ("tokens.scale", scale), ("tokens.sums", sums)):
        check_device(t, weight.device, what)
    dtype = out_dtype if out_dtype is not None else torch.bfloat16 if out is None else out.dtype
    if dtype not in DTYPE_CODES:
        raise ValueError(f"out_dtype must be bfloat16, float16 or float32, got {dtype}")
    ld = q.stride(0) if n > 1 else width
    with torch.cuda.device(weight.device):
        if ld % TOKEN_ALIGN or not width <= ld <= MAX_LD or q.data_ptr() % 16:
            q, ld = q[:, :width].clone(memory_format=torch.contiguous_format), width
        y, out_ld = _output(out, (*shape, weight.out_features), dtype, weight.device)
        _native.call("sh_matmul_i8", q.data_ptr(), ld, scale.data_ptr(), sums.data_ptr(), n, weight._ref, y.data_ptr(),
                     DTYPE_CODES[dtype], out_ld, current_stream_handle())
    if out is not None:
        increment_version(out)
    return y


def linear_i8(x: torch.Tensor, weight: Int8Weight, out: torch.Tensor | None = None,
              stream: torch.cuda.Stream | int | None = None) -> torch.Tensor:
    """``x · weightᵀ + bias`` in the type of ``x``, with the tokens of ``x`` quantised as
    :func:`quantize_tokens` does: the same values as the two calls, in fewer launches."""
    if stream is not None:
        with on_stream(stream, weight.qweight):
            return linear_i8(x, weight, out)
    code = _check_input(x, "linear_i8")
    index = weight.device.index
    if x.get_device() != index:
        raise ValueError(f"x must be on {weight.device}, got {x.device}")
    rows, tokens, ld = _token_rows(x, "x")
    if rows.shape[1] != weight.in_features:
        raise ValueError(f"x has {rows.shape[1]} values per token, the weight takes {weight.in_features}")
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            return linear_i8(x, weight, out)
    if out is None:
        out_ld = weight.out_features
        y = x.new_empty((*x.shape[:-1], out_ld))
    else:
        y, out_ld = _output(out, (*x.shape[:-1], weight.out_features), x.dtype, weight.device)
    lib = _native.lib()
    need = ctypes.c_uint64()
    _native.check(lib.sh_linear_i8_workspace(tokens, weight._ref, ctypes.byref(need)))
    ws = x.new_empty(need.value, dtype=torch.uint8) if need.value else None
    _native.check(lib.sh_linear_i8(rows.data_ptr(), code, ld, tokens, weight._ref, y.data_ptr(), out_ld,
                                   None if ws is None else ws.data_ptr(), need.value, current_stream_handle()))
    if out is not None:
        increment_version(out)
    return y
