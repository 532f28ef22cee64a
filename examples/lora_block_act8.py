"""A training step of a DiT block whose activations are kept in 8 bits: LoRA adapters, modulated norms, recomputation.

The block is the training DiT's of ``bench_workloads.py`` without its cross-attention: adaLN modulation, self-attention with
LoRA on q, k, v and o, a GELU MLP; base weights are frozen. Its norms keep their input in 8 bits
(``stagehand_amd.layer_norm``), the three LoRA A of q, k and v share one kept input (``stagehand_amd.act8``), and with
``--recompute`` the whole block is recomputed from its input, kept in 8 bits.

    python examples/lora_block_act8.py [--hidden 4096] [--heads 32] [--tokens 4096] [--rank 32] [--recompute]

runs a step with activations kept in 8 bits and one as torch keeps them, and prints how far the adapters' gradients are
apart, what the forward leaves in memory, and how long both take.
"""
from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

import torch
from torch import nn
from torch.nn import functional as F
from torch.nn.attention import SDPBackend, sdpa_kernel
from torch.utils.checkpoint import checkpoint

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from stagehand_amd.act8 import checkpoint_act8, linear_act8, quantize_activation  # noqa: E402
from stagehand_amd.layer_norm import layer_norm  # noqa: E402


class LoRA(nn.Module):
    """A frozen Linear and a trainable update of low rank: y = x Wᵀ + (x Aᵀ) Bᵀ."""

    def __init__(self, inp: int, out: int, rank: int, dtype: torch.dtype) -> None:
        super().__init__()
        self.weight = nn.Parameter(torch.empty(out, inp, device="cuda", dtype=dtype), requires_grad=False)
        self.a = nn.Parameter(torch.empty(rank, inp, device="cuda", dtype=dtype))
        self.b = nn.Parameter(torch.empty(out, rank, device="cuda", dtype=dtype))

    def forward(self, x: torch.Tensor, kept=None, keep8: bool = True) -> torch.Tensor:
        if not keep8:
            return F.linear(x, self.weight) + F.linear(F.linear(x, self.a), self.b)
        return F.linear(x, self.weight) + linear_act8(linear_act8(x, self.a, kept=kept), self.b)


class Block(nn.Module):
    def __init__(self, hidden: int, heads: int, rank: int, dtype: torch.dtype = torch.bfloat16, seed: int = 0) -> None:
        super().__init__()
        self.hidden, self.heads = hidden, heads
        self.q, self.k, self.v, self.o = (LoRA(hidden, hidden, rank, dtype) for _ in range(4))
        frozen = dict(modulation=(6 * hidden, hidden), up=(4 * hidden, hidden), down=(hidden, 4 * hidden))
        for name, shape in frozen.items():
            setattr(self, name, nn.Parameter(torch.empty(shape, device="cuda", dtype=dtype), requires_grad=False))
        g = torch.Generator(device="cuda").manual_seed(seed)
        with torch.no_grad():
            for p in self.parameters():
                p.copy_(torch.randn(p.shape, device="cuda", generator=g) * p.shape[1] ** -0.5)

    def adapters(self) -> list[nn.Parameter]:
        return [p for p in self.parameters() if p.requires_grad]

    def _norm(self, x: torch.Tensor, scale: torch.Tensor, shift: torch.Tensor, keep8: bool) -> torch.Tensor:
        if keep8:
            return layer_norm(x, scale, shift, modulate=True, keep8=True)
        return F.layer_norm(x, (self.hidden,), eps=1e-6) * (1 + scale) + shift

    def forward(self, x: torch.Tensor, vec: torch.Tensor, keep8: bool = True) -> torch.Tensor:
        b, s, h = x.shape
        m = F.linear(F.silu(vec), self.modulation)[:, None].chunk(6, dim=-1)
        xn = self._norm(x, m[1], m[0], keep8)
        kept = quantize_activation(xn.detach()) if keep8 and torch.is_grad_enabled() else None
        q, k, v = (p(xn, kept, keep8).view(b, s, self.heads, -1).transpose(1, 2).contiguous() for p in (self.q, self.k, self.v))
        with sdpa_kernel([SDPBackend.FLASH_ATTENTION, SDPBackend.EFFICIENT_ATTENTION]):
            a = F.scaled_dot_product_attention(q, k, v)
        x = x + m[2] * self.o(a.transpose(1, 2).reshape(b, s, h), keep8=keep8)
        xn = self._norm(x, m[4], m[3], keep8)
        return x + m[5] * F.linear(F.gelu(F.linear(xn, self.up), approximate="tanh"), self.down)


def step(block: Block, x: torch.Tensor, vec: torch.Tensor, dy: torch.Tensor, keep8: bool = True, recompute: bool = False):
    """(bytes that the forward keeps besides its output, gradients of x and the adapters)."""
    x = x.detach().requires_grad_()
    before = torch.cuda.memory_allocated()
    h = x * 1  # the block before: its output is the block's to keep
    if not recompute:
        y = block(h, vec, keep8)
    elif keep8:
        y = checkpoint_act8(block, h, vec)
    else:
        y = checkpoint(block, h, vec, False, use_reentrant=False)
    del h
    kept = torch.cuda.memory_allocated() - before - y.numel() * y.element_size()
    return kept, torch.autograd.grad(y, (x, *block.adapters()), dy)


def _time(f, n: int = 5) -> float:
    for _ in range(4):
        f()
    torch.cuda.synchronize()
    begin = time.perf_counter()
    for _ in range(n):
        f()
    torch.cuda.synchronize()
    return (time.perf_counter() - begin) / n * 1e3


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--hidden", type=int, default=4096)
    ap.add_argument("--heads", type=int, default=32)
    ap.add_argument("--tokens", type=int, default=4096)
    ap.add_argument("--rank", type=int, default=32)
    ap.add_argument("--recompute", action="store_true", help="recompute the block from its input")
    a = ap.parse_args()
    block = Block(a.hidden, a.heads, a.rank)
    g = torch.Generator(device="cuda").manual_seed(1)
    x, dy = (torch.randn(1, a.tokens, a.hidden, device="cuda", generator=g).bfloat16() for _ in range(2))
    vec = torch.randn(1, a.hidden, device="cuda", generator=g).bfloat16()
    results = {}
    for keep8 in (True, False):  # what libraries allocate and load once
        step(block, x, vec, dy, keep8, a.recompute)
    for keep8 in (True, False):
        kept, grads = step(block, x, vec, dy, keep8, a.recompute)
        results[keep8] = grads
        ms = _time(lambda: step(block, x, vec, dy, keep8, a.recompute))
        print(f"{'8 bits' if keep8 else 'torch '}: {kept / 1e6:.0f} MB kept, {ms:.2f} ms a step")
    far = [float((p.float() - q.float()).norm() / q.float().norm()) for p, q in zip(*results.values())]
    print(f"gradients apart: input {far[0]:.4f}, adapters {max(far[1:]):.4f} at most")


if __name__ == "__main__":
    main()
