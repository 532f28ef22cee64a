"""Timed cases of the operators on SquareQ weights and attention heads.

- ``linear``: ``stagehand_amd.int8.linear_i8``, a Linear layer on a SquareQ weight that stays in int8:
  the tokens are quantised to int8, one scale each, and multiplied with the int8 rows.
- ``qk``: ``stagehand_amd.qk_norm.qk_norm_rope``, RMS norm of every head of the queries and keys and the
  position rotation; ``train`` cases are the forward and the gradients of both inputs and both weights.

Where ``own`` is false, ``run`` computes the same in elementary torch operations, in 32 bits, rounded once.
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ── the cases ────────────────────────────────────────────────────────────────


def listed() -> list[dict]:
    return [
        # the smallest layer a test model streams (64-wide MLP block), a few tokens: latency of one call
        dict(name="lin_tiny", kind="linear", tokens=5, out=256, inp=64, pad=0, zp=False, bias=True, dtype="bf16"),
        # one token through a square projection of the 32-head training model: weight bytes
        dict(name="lin_token", kind="linear", tokens=1, out=4096, inp=4096, pad=0, zp=False, bias=True, dtype="bf16"),
        # the modulation of a DiT block for a batch of images, one conditioning row each: six hidden-sized outputs
        dict(name="lin_modulation", kind="linear", tokens=8, out=18432, inp=3072, pad=0, zp=False, bias=True, dtype="bf16"),
        # odd everything: short captions, a ragged layer with padded slab rows and zero points
        dict(name="lin_ragged", kind="linear", tokens=77, out=1000, inp=1155, pad=13, zp=True, bias=False, dtype="f16"),
        # the text stream's qkv projection
        dict(name="lin_text", kind="linear", tokens=512, out=9216, inp=3072, pad=0, zp=False, bias=True, dtype="bf16"),
        # a single-stream block's fused qkv + MLP projection over text and image tokens, padded rows with zero points
        dict(name="lin_stream", kind="linear", tokens=4608, out=21504, inp=3072, pad=16, zp=True, bias=True, dtype="bf16"),
        # the MLP's second Linear of the training model over a long video: the largest product
        dict(name="lin_video", kind="linear", tokens=16384, out=4096, inp=16384, pad=0, zp=False, bias=True, dtype="bf16"),
        # decoding: one new token for each of 16 sequences, grouped key heads, every sequence at its own position
        dict(name="qk_token", kind="qk", train=False, batch=16, seq=1, heads=32, kv=8, dim=128, rot=128,
             interleaved=False, positions=True, dtype="bf16"),
        # the joint text + image sequence of the 12B DiT
        dict(name="qk_stream", kind="qk", train=False, batch=1, seq=4608, heads=24, kv=24, dim=128, rot=128,
             interleaved=True, positions=False, dtype="bf16"),
        # odd lengths, a head size that is no power of two, a partial rotation
        dict(name="qk_ragged", kind="qk", train=False, batch=3, seq=1013, heads=10, kv=5, dim=80, rot=32,
             interleaved=False, positions=True, dtype="f16"),
        # a training step of a small float32 model
        dict(name="qk_train_small", kind="qk", train=True, batch=2, seq=257, heads=6, kv=6, dim=64, rot=64,
             interleaved=True, positions=False, dtype="f32"),
        # a training step of the 17.8B model's self-attention
        dict(name="qk_train", kind="qk", train=True, batch=2, seq=8192, heads=32, kv=32, dim=128, rot=128,
             interleaved=False, positions=False, dtype="bf16"),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    if rng.random() < 0.55:
        out, inp = _log_int(rng, 64, 21504), _log_int(rng, 64, 16384)
        if rng.random() < 0.6:  # widths as models have them, and any others
            out, inp = max(64, out // 64 * 64), max(64, inp // 64 * 64)
        most = min(16384, int(16384 * 4096 * 16384 / (out * inp)))
        return dict(kind="linear", tokens=_log_int(rng, 1, most), out=out, inp=inp, pad=rng.choice([0, 0, 3, 16]),
                    zp=rng.random() < 0.4, bias=rng.random() < 0.7, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]))
    dim = rng.choice([32, 64, 64, 72, 80, 96, 128, 128, 128, 256])
    heads = _log_int(rng, 1, 48)
    kv = rng.choice([d for d in range(1, heads + 1) if heads % d == 0])
    batch = _log_int(rng, 1, 32)
    most = 2 * 8192 * 64 * 128 // (batch * (heads + kv) * dim * 2)
    seq = 1 if rng.random() < 0.2 else _log_int(rng, 2, max(3, min(16384, most)))
    return dict(kind="qk", train=rng.random() < 0.5, batch=batch, seq=seq, heads=heads, kv=kv, dim=dim,
                rot=rng.choice([dim, dim, dim // 2 // 2 * 2]), interleaved=rng.random() < 0.5,
                positions=rng.random() < 0.5, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]))


# ── inputs ───────────────────────────────────────────────────────────────────


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, g) -> torch.Tensor:
    return torch.randn(shape, device="cuda", generator=g)


def _linear_inputs(c: dict, seed: int) -> dict:
    """Activations with a few strong channels and a padding token of zeros, and SquareQ rows."""
    g = _gen(seed)
    gain = torch.exp(0.7 * _randn((c["inp"],), g))
    x = _randn((c["tokens"], c["inp"]), g) * gain
    if c["tokens"] > 32:
        x[-1] = 0
    ld = c["inp"] + c["pad"]
    return dict(
        x=x.to(DTYPES[c["dtype"]]),
        q=torch.randint(-127, 128, (c["out"], ld), dtype=torch.int8, device="cuda", generator=g),
        scale=torch.exp(_randn((c["out"],), g) * 0.5 - 6.0),
        zero_point=_randn((c["out"],), g) if c["zp"] else None,
        bias=_randn((c["out"],), g) * 0.1 if c["bias"] else None,
    )


def _qk_inputs(c: dict, seed: int) -> dict:
    """Heads as a fused projection leaves them: (batch, seq, q heads + k heads + v heads, dim), seen as
    (batch, heads, seq, dim)."""
    g = _gen(seed)
    dt = DTYPES[c["dtype"]]
    b, s, hq, hk, d = c["batch"], c["seq"], c["heads"], c["kv"], c["dim"]
    qkv = (_randn((b, s, hq + 2 * hk, d), g) * 1.5).to(dt)
    rows = 4 * s + 64 if c["positions"] else s
    freq = 10000.0 ** (-torch.arange(c["rot"] // 2, device="cuda", dtype=torch.float64) * 2 / c["rot"])
    angle = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * freq
    state = dict(
        q=qkv[:, :, :hq].transpose(1, 2), k=qkv[:, :, hq:hq + hk].transpose(1, 2),
        q_weight=(1 + 0.1 * _randn((d,), g)).to(dt), k_weight=(1 + 0.1 * _randn((d,), g)).to(dt),
        cos=angle.cos().float(), sin=angle.sin().float(),
        positions=torch.randint(0, rows, (b, s), device="cuda", generator=g) if c["positions"] else None,
    )
    if c["train"]:
        state["dq_out"] = _randn((b, hq, s, d), g).to(dt)
        state["dk_out"] = _randn((b, hk, s, d), g).to(dt)
    return state


def prepare(case: dict, seed: int) -> dict:
    if case["kind"] == "linear":
        state = _linear_inputs(case, seed)
        if own:  # the handle that a program keeps for each layer
            from stagehand_amd.int8 import Int8Weight

            state["weight"] = Int8Weight(state["q"], state["scale"], zero_point=state["zero_point"], bias=state["bias"],
                                         in_features=case["inp"])
    else:
        state = _qk_inputs(case, seed)
        if case["train"]:
            for name in ("q", "k", "q_weight", "k_weight"):
                state[name] = state[name].detach().requires_grad_()
    state["case"] = case
    return state


# ── one pass ─────────────────────────────────────────────────────────────────


def run(state: dict):
    if own:
        return _own_linear(state) if state["case"]["kind"] == "linear" else _own_qk(state)
    with torch.no_grad():
        return _plain_linear(state) if state["case"]["kind"] == "linear" else _plain_qk(state)


def _own_linear(s: dict):
    from stagehand_amd.int8 import linear_i8

    return linear_i8(s["x"], s["weight"])


def _own_qk(s: dict):
    from stagehand_amd.qk_norm import qk_norm_rope

    q, k = qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], s["cos"], s["sin"], positions=s["positions"],
                        interleaved=s["case"]["interleaved"], eps=EPS)
    if not s["case"]["train"]:
        return {"q": q, "k": k}
    dq, dk, dqw, dkw = torch.autograd.grad((q, k), (s["q"], s["k"], s["q_weight"], s["k_weight"]),
                                           (s["dq_out"], s["dk_out"]))
    return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk, "dq_weight": dqw, "dk_weight": dkw}


def _plain_linear(s: dict):
    """y = (int8(x) · (Q − z)ᵀ) · token scale · row scale + bias, with int8(x) = rint(127 x / max |x|)."""
    x = s["x"].float()
    amax = x.abs().amax(1, keepdim=True)
    some = amax >= 2.0 ** -120
    inv = torch.where(some, torch.full_like(amax, 127.0) / amax, torch.zeros_like(amax))
    xs = torch.where(some, amax * (1.0 / 127.0), torch.zeros_like(amax))
    xq = torch.round(x * inv)
    w = s["q"][:, :x.shape[1]].float()
    if s["zero_point"] is not None:
        w = w - s["zero_point"][:, None]
    y = xq @ w.t() * xs * s["scale"]
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(s["x"].dtype)


def _tables(s: dict, seq: int):
    """cos and sin, (batch or 1, 1, seq, rot / 2)."""
    p = s["positions"]
    if p is None:
        return s["cos"][None, None, :seq], s["sin"][None, None, :seq]
    return s["cos"][p][:, None], s["sin"][p][:, None]


def _rotate(n, cos, sin, interleaved: bool):
    rot = 2 * cos.shape[-1]
    if interleaved:
        a, b = n[..., 0:rot:2], n[..., 1:rot:2]
        r = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = n[..., :rot // 2], n[..., rot // 2:rot]
        r = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((r, n[..., rot:]), -1) if rot < n.shape[-1] else r


def _plain_qk(s: dict):
    inter, out = s["case"]["interleaved"], {}
    cos, sin = _tables(s, s["case"]["seq"])
    for name in ("q", "k"):
        x, w = s[name].float(), s[name + "_weight"].float()
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        xn = x * r
        out[name] = _rotate(xn * w, cos, sin, inter).to(s[name].dtype)
        if s["case"]["train"]:
            g = _rotate(s[f"d{name}_out"].float(), cos, -sin, inter)
            h = g * w
            out["d" + name] = (r * (h - xn * (h * xn).mean(-1, keepdim=True))).to(s[name].dtype)
            out[f"d{name}_weight"] = (g * xn).sum((0, 1, 2)).to(s[name + "_weight"].dtype)
    return out


# ── what a pass cannot do without, and its results in 64 bits ────────────────


def work(case: dict) -> dict:
    c = case
    e = 4 if c["dtype"] == "f32" else 2
    if c["kind"] == "linear":
        m, n, k = c["tokens"], c["out"], c["inp"]
        return {"bytes": m * k * e + n * k + 4 * n * (1 + c["zp"] + c["bias"]) + m * n * e, "flops": 2.0 * m * n * k}
    values = c["batch"] * c["seq"] * (c["heads"] + c["kv"]) * c["dim"]
    table = 4 * c["seq"] * (c["batch"] if c["positions"] else 1) * c["rot"]
    if not c["train"]:
        return {"bytes": 2 * e * values + table, "flops": 9.0 * values}
    # forward: x in, y out; backward: x and dy in, dx out
    return {"bytes": 5 * e * values + 2 * table, "flops": 27.0 * values}


def exact(case: dict, seed: int):
    if case["kind"] == "linear":
        s = _linear_inputs(case, seed)
        x = s["x"].double()
        step = x.abs().max(1).values / 127
        q = torch.where(step[:, None] > 0, torch.round(x / step.clamp_min(1e-300)[:, None]), torch.zeros_like(x))
        w = s["q"][:, :case["inp"]].double()
        if s["zero_point"] is not None:
            w -= s["zero_point"].double()[:, None]
        w *= s["scale"].double()[:, None]
        y = (q * step[:, None]) @ w.t()
        return y if s["bias"] is None else y.add_(s["bias"].double())
    s = _qk_inputs(case, seed)
    d, rot = case["dim"], case["rot"]
    pos = s["positions"] if s["positions"] is not None else torch.arange(case["seq"], device="cuda")[None]
    c, t = s["cos"].double()[pos][:, None], s["sin"].double()[pos][:, None]
    # the pair of every rotated element, and the sign of the partner's share
    i = torch.arange(rot, device="cuda")
    if case["interleaved"]:
        pair, other, sign = i // 2, i ^ 1, 2.0 * (i % 2) - 1
    else:
        pair, other, sign = i % (rot // 2), (i + rot // 2) % rot, torch.where(i < rot // 2, -1.0, 1.0)
    out = {}
    for name in ("q", "k"):
        x = s[name].double().requires_grad_()
        w = s[name + "_weight"].double().requires_grad_()
        with torch.enable_grad():
            n = w * x / (x.square().sum(-1, keepdim=True) / d + EPS).sqrt()
            rotated = n[..., :rot] * c[..., pair] + n[..., other] * (t[..., pair] * sign)
            y = torch.cat((rotated, n[..., rot:]), -1)
            if case["train"]:
                dx, dw = torch.autograd.grad(y, (x, w), s[f"d{name}_out"].double())
                out["d" + name], out[f"d{name}_weight"] = dx, dw
        out[name] = y.detach()
    return out
