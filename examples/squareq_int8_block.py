"""A DiT single-stream block on SquareQ weights that stay in int8, and a training step of its norms.

The block's Linears come from a SquareQ V2 slab (safetensors + manifest, as ``read_v2_layers`` gives
them) and are multiplied as they are (``stagehand_amd.int8``); queries and keys are normed and rotated
in one pass (``stagehand_amd.qk_norm``), forward and backward. The layout is the single-stream block of
``bench_workloads.py``, with a rotary position embedding.

    python examples/squareq_int8_block.py [--hidden 3072] [--heads 24] [--tokens 4608]

writes a slab with random weights, runs the block on it and on the dequantised weights, and prints
how far the results are apart and how long both take.
"""
from __future__ import annotations

import argparse
import sys
import tempfile
import time
from pathlib import Path

import torch
from torch import nn
from torch.nn import functional as F
from torch.nn.attention import SDPBackend, sdpa_kernel

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from stagehand_amd.int8 import Int8Weight, linear_i8  # noqa: E402
from stagehand_amd.qk_norm import qk_norm_rope  # noqa: E402
from stagehand_amd.squareq_v2 import read_v2_layers, write_v2_slab  # noqa: E402

LINEARS = ("modulation", "linear1", "linear2")


def linear_shapes(hidden: int, mlp: int) -> dict[str, tuple[int, int]]:
    return {"modulation": (3 * hidden, hidden), "linear1": (3 * hidden + mlp, hidden), "linear2": (hidden, hidden + mlp)}


def write_slab(path: str, hidden: int, mlp: int, seed: int = 0) -> str:
    """A slab of the block's Linears: int8 rows of N(0, 1 / inputs) weights, one scale each. Returns its manifest."""
    g = torch.Generator().manual_seed(seed)
    layers = {}
    for name, (out_f, in_f) in linear_shapes(hidden, mlp).items():
        w = torch.randn(out_f, in_f, generator=g) * in_f ** -0.5
        scale = w.abs().amax(1) / 127
        layers[name] = {"qweight": torch.round(w / scale[:, None]).to(torch.int8), "scale": scale,
                        "bias": torch.randn(out_f, generator=g) * 0.02}
    return write_v2_slab(path, layers)


def rotary_tables(tokens: int, dim: int, device: str = "cuda") -> tuple[torch.Tensor, torch.Tensor]:
    freq = 10000.0 ** (-torch.arange(dim // 2, dtype=torch.float64) * 2 / dim)
    angle = torch.arange(tokens, dtype=torch.float64)[:, None] * freq
    return angle.cos().float().to(device), angle.sin().float().to(device)


class SingleStreamBlock(nn.Module):
    """``linears``: name → a function of the activations, an int8 product or any other Linear."""

    def __init__(self, linears: dict, hidden: int, heads: int, mlp: int) -> None:
        super().__init__()
        self.linears, self.hidden, self.heads, self.mlp = linears, hidden, heads, mlp
        self.q_weight = nn.Parameter(torch.ones(hidden // heads, device="cuda", dtype=torch.bfloat16))
        self.k_weight = nn.Parameter(torch.ones(hidden // heads, device="cuda", dtype=torch.bfloat16))

    def forward(self, x: torch.Tensor, vec: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
        h, b, s = self.hidden, x.shape[0], x.shape[1]
        shift, scale, gate = self.linears["modulation"](F.silu(vec))[:, None, :].chunk(3, dim=-1)
        xn = F.layer_norm(x, (h,), eps=1e-6) * (1 + scale) + shift
        qkv, mlp_in = torch.split(self.linears["linear1"](xn), [3 * h, self.mlp], dim=-1)
        q, k, v = (t.transpose(1, 2) for t in qkv.unflatten(-1, (3, self.heads, h // self.heads)).unbind(2))
        q, k = qk_norm_rope(q, k, self.q_weight, self.k_weight, cos, sin, interleaved=True)
        with sdpa_kernel([SDPBackend.FLASH_ATTENTION, SDPBackend.EFFICIENT_ATTENTION]):
            attn = F.scaled_dot_product_attention(q, k, v.contiguous()).transpose(1, 2).reshape(b, s, h)
        return x + gate * self.linears["linear2"](torch.cat([attn, F.gelu(mlp_in, approximate="tanh")], dim=-1))


def int8_linears(layers: dict, shapes: dict) -> dict:
    weights = {n: Int8Weight.from_squareq(layers[n], *shapes[n]) for n in shapes}
    return {n: (lambda x, w=w: linear_i8(x, w)) for n, w in weights.items()}


def dequantised_linears(layers: dict, shapes: dict) -> dict:
    out = {}
    for n, (out_f, in_f) in shapes.items():
        w = Int8Weight.from_squareq(layers[n], out_f, in_f)
        out[n] = lambda x, w=w.dequantize(torch.bfloat16), b=w.bias.to(torch.bfloat16): F.linear(x, w, b)
    return out


def load(path: str, manifest: str, hidden: int, heads: int, mlp: int) -> tuple[SingleStreamBlock, SingleStreamBlock]:
    """The block on the slab's int8 rows, and on their dequantised values."""
    view = memoryview(bytearray(Path(path).read_bytes()))
    layers, shapes = read_v2_layers(path, manifest, view), linear_shapes(hidden, mlp)
    return (SingleStreamBlock(int8_linears(layers, shapes), hidden, heads, mlp),
            SingleStreamBlock(dequantised_linears(layers, shapes), hidden, heads, mlp))


def train_norms(block: SingleStreamBlock, x: torch.Tensor, vec: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                target: torch.Tensor, steps: int, lr: float) -> list[float]:
    """Fits the block's norm weights to ``target`` by gradient descent; the losses before each step."""
    losses = []
    for _ in range(steps):
        loss = (block(x, vec, cos, sin).float() - target.float()).square().mean()
        grads = torch.autograd.grad(loss, (block.q_weight, block.k_weight))
        with torch.no_grad():
            for w, g in zip((block.q_weight, block.k_weight), grads):
                w -= lr * g
        losses.append(float(loss.detach()))
    return losses


def _time(f, n: int = 10) -> float:
    f()
    torch.cuda.synchronize()
    begin = time.perf_counter()
    for _ in range(n):
        f()
    torch.cuda.synchronize()
    return (time.perf_counter() - begin) / n * 1e3


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--hidden", type=int, default=3072)
    ap.add_argument("--heads", type=int, default=24)
    ap.add_argument("--tokens", type=int, default=4608)
    a = ap.parse_args()
    mlp = 4 * a.hidden
    with tempfile.TemporaryDirectory() as tmp:
        path = str(Path(tmp) / "block.safetensors")
        manifest = write_slab(path, a.hidden, mlp)
        block, plain = load(path, manifest, a.hidden, a.heads, mlp)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(1, a.tokens, a.hidden, device="cuda", generator=g).to(torch.bfloat16)
    vec = torch.randn(1, a.hidden, device="cuda", generator=g).to(torch.bfloat16)
    cos, sin = rotary_tables(a.tokens, a.hidden // a.heads)
    with torch.no_grad():
        y, want = block(x, vec, cos, sin), plain(x, vec, cos, sin)
        far = float((y - want).float().norm() / (want - x).float().norm())
        print(f"int8 against dequantised: {far:.4f} of the block's update")
        print(f"int8 {_time(lambda: block(x, vec, cos, sin)):.3f} ms, dequantised {_time(lambda: plain(x, vec, cos, sin)):.3f} ms")


if __name__ == "__main__":
    main()
