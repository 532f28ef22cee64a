"""The 8-bit format of activations in 64 bits: groups of 32 features, a power of two for each, whole multiples of it."""
from __future__ import annotations

import torch

ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # half a step, relative
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -149}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
GROUP = 32


def quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(q as int8, exponent bytes) of the rows of a 2-D tensor, on the CPU. Exact: every product is by a power of two."""
    tokens, cols = x.shape
    groups = -(-cols // GROUP)
    v = torch.zeros(tokens, groups * GROUP, dtype=torch.float64)
    v[:, :cols] = x.detach().cpu().double()
    v = v.view(tokens, groups, GROUP)
    broken = ~v.isfinite().all(-1)
    top = v.abs().amax(-1)
    m, e = torch.frexp(torch.where(broken, torch.zeros_like(top), top))  # top = m 2^e, 1/2 <= m < 1
    k = torch.where(m <= 127 / 128, e - 7, e - 6).clamp_min(-126)
    k = torch.where(m == 0, torch.full_like(k, -126), k)
    step = torch.pow(torch.tensor(2.0, dtype=torch.float64), k.double())
    assert bool((torch.frexp(step)[0] == 0.5).all())  # powers of two indeed
    q = torch.round(v / step[..., None])
    most = torch.where(k == (10 if x.dtype == torch.float16 else 122), 63.0, 127.0).double()[..., None]
    q = torch.where(broken[..., None], torch.zeros_like(q), torch.minimum(torch.maximum(q, -most), most))
    return q.to(torch.int8).view(tokens, groups * GROUP), torch.where(broken, torch.full_like(k, 255), k + 127).to(torch.uint8)


def dequantize(q: torch.Tensor, exponent: torch.Tensor, cols: int) -> torch.Tensor:
    """The kept values in 64 bits, on the CPU."""
    q, exponent = q.cpu(), exponent.cpu()
    step = torch.pow(torch.tensor(2.0, dtype=torch.float64), exponent.double() - 127)
    step = torch.where(exponent == 255, torch.full_like(step, float("nan")), step)
    return (q.view(*exponent.shape, GROUP).double() * step[..., None]).flatten(-2)[..., :cols]


def kept_values(x: torch.Tensor) -> torch.Tensor:
    """What is read back of a 2-D tensor, in 64 bits, on the CPU."""
    return dequantize(*quantize(x), x.shape[1])


def activations(*shape: int, dtype: torch.dtype = torch.float32, seed: int = 0) -> torch.Tensor:
    """Features of different strength, off zero."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    cols = shape[-1]
    gain = torch.exp(0.7 * torch.randn(cols, device="cuda", generator=g))
    return (torch.randn(shape, device="cuda", generator=g) * gain + 0.3 * torch.randn(cols, device="cuda", generator=g)).to(dtype)
