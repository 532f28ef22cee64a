"""RMS norms of query and key heads with the position rotation, in one pass, with gradients.

For every head of the queries and keys::

    n = x * weight * rsqrt(mean(x²) + eps)
    out[a], out[b] = n[a] c - n[b] s, n[b] c + n[a] s        for the rot / 2 pairs (a, b)

with ``(a, b) = (p, p + rot / 2)``, or ``(2p, 2p + 1)`` when ``interleaved``, and ``c, s`` the row of
the tables ``cos`` and ``sin`` that belongs to the token's position. Statistics, products and the
weights' gradients are held in fp32; outputs and gradients are rounded once.

Everything runs on the caller's current torch stream unless ``stream`` is given. There is no CPU path.
"""
from __future__ import annotations

import ctypes
import struct

import torch
from torch.autograd.graph import increment_version

from stagehand_amd import _native
from stagehand_amd.int8 import DTYPE_CODES, check_no_grad, check_no_tangent, on_stream
from stagehand_amd.unpack import current_stream_handle

__all__ = ["qk_norm_rope"]

MAX_DIM = 512  # SH_QK_MAX_DIM

# Mirror of `struct sh_qk_norm_rope_args`: six sh_heads, then pointers and strides, then 32-bit fields.
_ARGS = struct.Struct("<24Q" "7Q" "2Q" "q" "11If")


_NO_HEADS = (0, 0, 0, 0)


def _heads(t: torch.Tensor | None) -> tuple[int, int, int, int]:
    if t is None:
        return _NO_HEADS
    b, h, s, _ = t.stride()
    return t.data_ptr(), b, h, s


def _ptr(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


def _rows_of_values(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(3) == 1 else t.contiguous()


def _fields(x, q_heads, k_heads, weight, cos, positions, start, interleaved, eps) -> tuple:
    """The struct's fields from table_ld on, for heads like those of ``x``."""
    batch, _, seq, dim = x.shape
    code = DTYPE_CODES[x.dtype]
    if cos is None:
        table_rows = half_rot = table_ld = start = 0
    else:
        table_rows, half_rot = cos.shape
        table_ld = cos.stride(0)
    if positions is None:
        position_stride = position_bytes = 0
    else:
        position_stride, position_bytes = positions.stride(0) if positions.dim() == 2 else 0, positions.element_size()
    return (table_ld, position_stride, start, table_rows, position_bytes, batch, seq, q_heads, k_heads, dim, 2 * half_rot,
            code, code if weight is None else DTYPE_CODES[weight.dtype], interleaved, eps)


def _run(q, k, q_weight, k_weight, cos, sin, positions, start, interleaved, eps, q_out, k_out):
    fields = _fields(q, q.shape[1], 0 if k is None else k.shape[1], k_weight if q_weight is None else q_weight, cos, positions,
                     start, interleaved, eps)
    args = _ARGS.pack(*_heads(q), *_heads(k), *_heads(q_out), *_heads(k_out), *_NO_HEADS, *_NO_HEADS, _ptr(q_weight),
                      _ptr(k_weight), 0, 0, _ptr(cos), _ptr(sin), _ptr(positions), *fields)
    _native.check(_native.lib().sh_qk_norm_rope(args, current_stream_handle()))


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, start, interleaved, eps):
        q_out = q.new_empty(q.shape)
        k_out = None if k is None else k.new_empty(k.shape)
        _run(q, k, q_weight, k_weight, cos, sin, positions, start, interleaved, eps, q_out, k_out)
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.options = start, interleaved, eps
        return q_out, k_out

    @staticmethod
    def backward(ctx, dq_out, dk_out):
        if torch.is_grad_enabled():  # create_graph
            raise RuntimeError("qk_norm_rope has no second derivatives")
        q, k, q_weight, k_weight, cos, sin, positions = ctx.saved_tensors
        want_q, want_k, want_qw, want_kw = ctx.needs_input_grad[:4]
        if want_q or want_qw:
            dq_out = _rows_of_values(dq_out)
        else:
            q = dq_out = None
        if want_k or want_kw:
            dk_out = _rows_of_values(dk_out)
        else:
            k = dk_out = None
        dq = _like(q) if want_q else None
        dk = _like(k) if want_k else None
        dqw = torch.empty_like(q_weight) if want_qw else None
        dkw = torch.empty_like(k_weight) if want_kw else None
        fields = _fields(k if q is None else q, 0 if q is None else q.shape[1], 0 if k is None else k.shape[1],
                         k_weight if q_weight is None else q_weight, cos, positions, *ctx.options)
        args = _ARGS.pack(*_heads(q), *_heads(k), *_heads(dq_out), *_heads(dk_out), *_heads(dq), *_heads(dk),
                          _ptr(q_weight), _ptr(k_weight), _ptr(dqw), _ptr(dkw), _ptr(cos), _ptr(sin), _ptr(positions), *fields)
        lib = _native.lib()
        ws, need = None, ctypes.c_uint64()
        if want_qw or want_kw:
            _native.check(lib.sh_qk_norm_rope_workspace(args, ctypes.byref(need)))
            ws = torch.empty(need.value, dtype=torch.uint8, device=(q if q is not None else k).device)
        _native.check(lib.sh_qk_norm_rope_backward(args, _ptr(ws), need.value, current_stream_handle()))
        return dq, dk, dqw, dkw, None, None, None, None, None, None


def _check_weight(w: torch.Tensor, what: str, device: int, dim: int) -> None:
    if w.get_device() != device or w.shape != (dim,) or w.dtype not in DTYPE_CODES or w.stride(0) != 1:
        raise ValueError(f"{what} must be {dim} contiguous values in bfloat16, float16 or float32 on q's device, "
                         f"got {w.device} {w.dtype} {tuple(w.shape)}")


def _like(x: torch.Tensor) -> torch.Tensor:
    """A tensor for the gradient of ``x``, with its dims in the order of ``x``'s memory."""
    d = torch.empty_like(x)
    return d if d.stride(3) == 1 else torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _heads_overlap(t: torch.Tensor) -> bool:
    """Whether heads of ``t`` may share memory: some distance between heads is less than what lies within it.
    (Slices, permutations and windows of a dense tensor never do.)"""
    if t.numel() == 0:
        return False
    reach = t.shape[3]
    for stride, size in sorted(zip(t.stride()[:3], t.shape)):
        if size > 1:
            if stride < reach:
                return True
            reach += (size - 1) * stride
    return False


def qk_norm_rope(
    q: torch.Tensor,
    k: torch.Tensor | None,
    q_weight: torch.Tensor | None = None,
    k_weight: torch.Tensor | None = None,
    cos: torch.Tensor | None = None,
    sin: torch.Tensor | None = None,
    *,
    positions: torch.Tensor | None = None,
    start: int = 0,
    interleaved: bool = False,
    eps: float = 1e-6,
    out: tuple[torch.Tensor, torch.Tensor | None] | None = None,
    stream: torch.cuda.Stream | int | None = None,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Normed and rotated ``(q, k)``; see the module's formulas.

    ``q`` is ``(batch, heads, seq, dim)``, ``k`` the same with any number of heads (or None). Any
    strides: views of a fused projection are read in place. ``q_weight`` and ``k_weight`` hold ``dim``
    values of one type, None stands for ones. ``cos`` and ``sin`` are float32 ``(positions, rot / 2)``
    with ``rot <= dim``; without them there is only the norm. Token ``s`` is at position ``start + s``,
    or at ``positions[s]`` / ``positions[b, s]`` (int32 or int64 on the device; a position that the
    tables do not have gives NaN for that token).

    The outputs are contiguous, or written to ``out``: tensors of the same shapes with any strides
    that keep a head's values together (a slice of a joint sequence, or ``q`` and ``k`` themselves, but no
    other memory of the inputs'). A backward pass that needs the old values of ``out`` raises.
    Gradients flow to ``q``, ``k`` and the weights, not to the tables, and not through ``out``."""
    if stream is not None:
        with on_stream(stream, q):
            return qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions=positions, start=start,
                                interleaved=interleaved, eps=eps, out=out)
    device, shape, dtype = q.get_device(), q.shape, q.dtype
    if device < 0 or len(shape) != 4 or dtype not in DTYPE_CODES:
        raise ValueError("q must be a device tensor (batch, heads, seq, dim) in bfloat16, float16 or float32, "
                         f"got {q.device} {dtype} {tuple(shape)}")
    batch, _, seq, dim = shape
    if dim % 2 or not 2 <= dim <= MAX_DIM:
        raise ValueError(f"dim {dim} is not an even number in 2 .. {MAX_DIM}")
    if k is not None:
        ks = k.shape
        if k.get_device() != device or k.dtype != dtype or len(ks) != 4 or ks[0] != batch or ks[2] != seq or ks[3] != dim:
            raise ValueError(f"k must be {dtype} on q's device with q's batch, seq and dim, got {k.device} {k.dtype} {tuple(ks)} "
                             f"for q {q.device} {tuple(shape)}")
    elif k_weight is not None:
        raise ValueError("k_weight is given without k")
    if q_weight is not None:
        _check_weight(q_weight, "q_weight", device, dim)
    if k_weight is not None:
        _check_weight(k_weight, "k_weight", device, dim)
        if q_weight is not None and q_weight.dtype != k_weight.dtype:
            raise ValueError(f"q_weight and k_weight must have one type, got {q_weight.dtype} and {k_weight.dtype}")
    if not 0.0 <= eps <= 1e38:
        raise ValueError(f"eps {eps} is negative or not finite")
    check_no_tangent("qk_norm_rope", q, k, q_weight, k_weight, cos, sin)
    grad_mode = torch.is_grad_enabled()
    if cos is not None and sin is not None:
        table = cos.shape
        if cos.get_device() != device or sin.get_device() != device or len(table) != 2 or sin.shape != table or \
                cos.dtype != torch.float32 or sin.dtype != torch.float32 or 2 * table[1] > dim or \
                cos.stride() != sin.stride() or (table[1] > 1 and cos.stride(1) != 1):
            raise ValueError(f"cos and sin must be float32 (positions, rot / 2) rows on q's device with rot <= {dim}, got "
                             f"{cos.device} {cos.dtype} {tuple(table)} and {sin.device} {sin.dtype} {tuple(sin.shape)}")
        if grad_mode and (cos.requires_grad or sin.requires_grad):
            raise ValueError("cos and sin have no gradient: detach them")
        if positions is None and not 0 <= start <= table[0] - seq:
            raise ValueError(f"positions {start} .. {start + seq - 1} are not all in the tables' {table[0]} rows")
        if table[1] == 0:
            cos = sin = None
    elif cos is not sin:
        raise ValueError("cos and sin are given together or not at all")
    if positions is not None:
        if cos is None or start:
            raise ValueError("positions are given with cos and sin, and without start")
        ps = tuple(positions.shape)
        if positions.get_device() != device or positions.dtype not in (torch.int64, torch.int32) or \
                ps not in ((batch, seq), (seq,), (1, seq)):
            raise ValueError(f"positions must be int32 or int64 ({seq},) or ({batch}, {seq}) on q's device, got "
                             f"{positions.device} {positions.dtype} {ps}")
        if len(ps) == 2 and ps[0] == 1:
            positions = positions[0]
        if seq > 1 and positions.stride(-1) != 1:
            positions = positions.contiguous()
    if device != torch.cuda.current_device():
        with torch.cuda.device(device):
            return qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions=positions, start=start,
                                interleaved=interleaved, eps=eps, out=out)
    q = _rows_of_values(q)
    k = None if k is None else _rows_of_values(k)
    grad = grad_mode and any([t is not None and t.requires_grad for t in (q, k, q_weight, k_weight)])
    if out is None:
        if grad:
            return _QkNormRope.apply(q, k, q_weight, k_weight, cos, sin, positions, start, bool(interleaved), eps)
        q_out = q.new_empty(shape)
        k_out = None if k is None else k.new_empty(k.shape)
    else:
        if grad:
            raise RuntimeError("out= has no gradient: call qk_norm_rope under torch.no_grad(), or without out")
        q_out, k_out = out
        for what, o, x in (("q", q_out, q), ("k", k_out, k)):
            if (o is None) != (x is None):
                raise ValueError(f"out has {'no' if o is None else 'a'} tensor for {what}")
            if o is None:
                continue
            if o.get_device() != device or o.shape != x.shape or o.dtype != dtype or o.stride(3) != 1:
                raise ValueError(f"out for {what} must be {dtype} {tuple(x.shape)} with contiguous heads on q's device, "
                                 f"got {o.device} {o.dtype} {tuple(o.shape)} strides {o.stride()}")
            if _heads_overlap(o):
                raise ValueError(f"heads of out for {what} share memory: {tuple(o.shape)} with strides {o.stride()}")
            check_no_grad(o, f"out for {what}")
            check_no_tangent(f"out for {what}", o)
    _run(q, k, q_weight, k_weight, cos, sin, positions, start, interleaved, eps, q_out, k_out)
    if out is not None:
        increment_version([o for o in (q_out, k_out) if o is not None])
    return q_out, k_out
