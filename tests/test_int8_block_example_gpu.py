"""The int8 block of examples/: its result against the same block on dequantised weights in float64, its norms
trained through the fused forward and backward, and its command."""
from __future__ import annotations

import importlib.util
import subprocess
import sys
from pathlib import Path

import pytest
import torch
from torch.nn import functional as F

REPO = Path(__file__).resolve().parent.parent
pytestmark = pytest.mark.gpu


def example():
    spec = importlib.util.spec_from_file_location("squareq_int8_block", REPO / "examples" / "squareq_int8_block.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def reference(layers, shapes, x, vec, cos, sin, heads, mlp):
    """The block in float64 on the CPU, on the dequantised weights."""
    x, vec, c, s = (t.double().cpu() for t in (x, vec, cos, sin))
    h = x.shape[-1]

    def lin(n, v):
        o, i = shapes[n]
        w = layers[n]["qweight"][:o, :i].double() * layers[n]["scale"].double()[:, None]
        return v @ w.t() + layers[n]["bias"].double()

    shift, scale, gate = lin("modulation", F.silu(vec))[:, None, :].chunk(3, -1)
    qkv, m = torch.split(lin("linear1", F.layer_norm(x, (h,), eps=1e-6) * (1 + scale) + shift), [3 * h, mlp], -1)
    q, k, v = (t.transpose(1, 2) for t in qkv.unflatten(-1, (3, heads, h // heads)).unbind(2))

    def norm(t):
        t = t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt()
        a, b = t[..., 0::2], t[..., 1::2]
        return torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)

    p = torch.softmax(norm(q) @ norm(k).transpose(-1, -2) * (h // heads) ** -0.5, -1)
    attn = (p @ v).transpose(1, 2).reshape(x.shape)
    return x + gate * lin("linear2", torch.cat([attn, F.gelu(m, approximate="tanh")], -1))


@pytest.mark.parametrize("hidden,heads,tokens", [(256, 4, 100), (192, 2, 33)])
def test_block_matches_the_dequantised_one(tmp_path, hidden, heads, tokens):
    """Each of the two products on the way to the output rounds its activations to 1 / 127 of a token's largest value,
    about 4 of its root mean squares: an error of 4 / 127 / sqrt(12) = 0.9% of the product each, and bfloat16's
    0.2% of each of some six steps: under 3% of the block's update."""
    ex = example()
    mlp = 4 * hidden
    path = str(tmp_path / "block.safetensors")
    manifest = ex.write_slab(path, hidden, mlp)
    block, plain = ex.load(path, manifest, hidden, heads, mlp)
    x = torch.randn(2, tokens, hidden, device="cuda").to(torch.bfloat16)
    vec = torch.randn(2, hidden, device="cuda").to(torch.bfloat16)
    cos, sin = ex.rotary_tables(tokens, hidden // heads)
    layers = ex.read_v2_layers(path, manifest, memoryview(bytearray(Path(path).read_bytes())))
    want = reference(layers, ex.linear_shapes(hidden, mlp), x, vec, cos, sin, heads, mlp)
    update = (want - x.double().cpu()).norm()
    with torch.no_grad():
        for b, most in ((block, 0.03), (plain, 0.015)):
            assert (b(x, vec, cos, sin).double().cpu() - want).norm() <= most * update


def test_norm_weights_train(tmp_path):
    ex = example()
    hidden, heads, mlp, tokens = 128, 2, 512, 40
    path = str(tmp_path / "block.safetensors")
    _, plain = ex.load(path, ex.write_slab(path, hidden, mlp), hidden, heads, mlp)
    x = torch.randn(1, tokens, hidden, device="cuda").to(torch.bfloat16)
    vec = torch.randn(1, hidden, device="cuda").to(torch.bfloat16)
    cos, sin = ex.rotary_tables(tokens, hidden // heads)
    with torch.no_grad():
        plain.q_weight.mul_(3.0)  # sharper attention, to be found again
        target = plain(x, vec, cos, sin)
        plain.q_weight.div_(3.0)
    # of the loss's own size, whatever the weights' draw: a step that moves the weights by a tenth
    loss = (plain(x, vec, cos, sin).float() - target.float()).square().mean()
    g = torch.autograd.grad(loss, (plain.q_weight,))[0].float()
    lr = 0.1 * float(plain.q_weight.detach().float().norm() / g.norm())
    losses = ex.train_norms(plain, x, vec, cos, sin, target, 8, lr)
    assert losses[-1] < losses[0]


def test_command():
    run = subprocess.run([sys.executable, str(REPO / "examples" / "squareq_int8_block.py"), "--hidden", "256", "--heads", "4",
                          "--tokens", "64"], capture_output=True, text=True, timeout=110)
    assert run.returncode == 0, run.stderr
    assert "int8 against dequantised: 0.0" in run.stdout
