"""Timed cases of layer norms, activations kept in 8 bits and the weight gradients that read them.

- ``norm``: ``stagehand_amd.layer_norm.layer_norm``, with a weight and a bias for all tokens or, ``modulate``, a
  scale and a shift for every sequence; ``train`` cases are the forward and the gradients of all three inputs, from the
  input itself or, ``keep8``, from what is kept of it in 8 bits.
- ``keep``: ``stagehand_amd.act8.quantize_activation`` and ``Activation8.dequantize``: an activation is written in
  8 bits, as a checkpoint, and read back.
- ``wgrad``: ``stagehand_amd.act8.weight_grad_act8``, the gradient of a Linear's weight (and bias) from its kept input.

What is kept: 32 neighbouring features share a power of two, the smallest 2^k with max |x| <= 127 * 2^k (k from -126 on),
and are rounded to whole multiples of it, ties to even; 63 of them at most where 64 would leave the type's range.

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
        # the norm of a small test block (hidden 64), a dozen tokens: latency of one call
        dict(name="norm_small", kind="norm", train=False, keep8=False, modulate=False, batch=1, seq=12, cols=64, dtype="f32"),
        # an image's and its caption's tokens through a modulated norm of the 4096-wide DiT, inference
        dict(name="norm_stream", kind="norm", train=False, keep8=False, modulate=True, batch=1, seq=4608, cols=4096, dtype="bf16"),
        # odd everything: a training step of a norm with weight and bias, rows off vector boundaries
        dict(name="norm_train_ragged", kind="norm", train=True, keep8=False, modulate=False, batch=3, seq=1013, cols=1155, dtype="f16"),
        # two long sequences through a modulated norm, training: gradients of scale and shift for each of them
        dict(name="norm_train", kind="norm", train=True, keep8=False, modulate=True, batch=2, seq=8192, cols=4096, dtype="bf16"),
        # the same kind of step where memory is short: the norm's input is kept in 8 bits for the backward pass
        dict(name="norm_train_kept", kind="norm", train=True, keep8=True, modulate=True, batch=4, seq=4096, cols=5120, dtype="bf16"),
        # a short caption's activations, ragged groups, written and read back: latency of two calls
        dict(name="keep_ragged", kind="keep", tokens=77, cols=1155, dtype="f32"),
        # the input of a block of the 4096-wide training DiT, written as a checkpoint and read for the recomputation
        dict(name="keep_block", kind="keep", tokens=8192, cols=4096, dtype="bf16"),
        # the first Linear of a small test block trained in fp32: latency
        dict(name="wgrad_small", kind="wgrad", tokens=77, out=256, inp=64, bias=True, dtype="f32"),
        # the LoRA A of an attention projection, rank 32, in the 4096-wide training DiT: one read of the kept input
        dict(name="wgrad_lora", kind="wgrad", tokens=4096, out=32, inp=4096, bias=False, dtype="bf16"),
        # odd everything
        dict(name="wgrad_ragged", kind="wgrad", tokens=1013, out=1000, inp=1155, bias=True, dtype="f16"),
        # an attention projection trained in full
        dict(name="wgrad_proj", kind="wgrad", tokens=4608, out=4096, inp=4096, bias=False, dtype="bf16"),
        # the wide Linear of an MLP trained in full, a long batch
        dict(name="wgrad_mlp", kind="wgrad", tokens=16384, out=16384, inp=4096, bias=True, dtype="bf16"),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["norm", "norm", "keep", "wgrad", "wgrad"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "norm":
        cols = _log_int(rng, 16, 16384)
        if rng.random() < 0.6:  # widths as models have them, and any others
            cols = max(64, cols // 64 * 64)
        batch = _log_int(rng, 1, 16)
        most = min(16384, 2 * 8192 * 4096 // (batch * cols))
        return dict(kind=kind, train=rng.random() < 0.65, keep8=rng.random() < 0.4, modulate=rng.random() < 0.5, batch=batch,
                    seq=1 if rng.random() < 0.15 else _log_int(rng, 1, max(2, most)), cols=cols, dtype=dtype)
    if kind == "keep":
        cols = _log_int(rng, 16, 16384)
        if rng.random() < 0.6:
            cols = max(64, cols // 64 * 64)
        return dict(kind=kind, tokens=_log_int(rng, 1, min(65536, 8192 * 8192 // cols)), cols=cols, dtype=dtype)
    out, inp = _log_int(rng, 8, 16384), _log_int(rng, 16, 16384)
    if rng.random() < 0.6:
        out, inp = max(8, out // 8 * 8), max(64, inp // 64 * 64)
    most = min(16384, 16384 * 4096 * 4096 // (out * inp))
    return dict(kind=kind, tokens=_log_int(rng, 1, most), out=out, inp=inp, bias=rng.random() < 0.5, dtype=dtype)


# ── inputs ───────────────────────────────────────────────────────────────────


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, g) -> torch.Tensor:
    return torch.randn(shape, device="cuda", generator=g)


def _activations(shape, dt, g) -> torch.Tensor:
    """Features of different strength, some strong ones among them, off zero; a padding token of zeros in long inputs."""
    cols = shape[-1]
    x = _randn(shape, g) * torch.exp(0.7 * _randn((cols,), g)) + 0.3 * _randn((cols,), g)
    if shape[-2] > 32:
        x[..., -1, :] = 0
    return x.to(dt)


def _inputs(c: dict, seed: int) -> dict:
    g, dt = _gen(seed), DTYPES[c["dtype"]]
    if c["kind"] == "keep":
        return dict(x=_activations((c["tokens"], c["cols"]), dt, g))
    if c["kind"] == "wgrad":
        return dict(x=_activations((c["tokens"], c["inp"]), dt, g), dy=(0.1 * _randn((c["tokens"], c["out"]), g)).to(dt))
    b, s, n = c["batch"], c["seq"], c["cols"]
    state = dict(x=_activations((b, s, n), dt, g))
    if c["modulate"]:  # what a block's modulation gives: six rows a sequence, of which a norm takes two
        six = (0.3 * _randn((b, 1, 6 * n), g)).to(dt).chunk(6, -1)
        state["weight"], state["bias"] = six[1], six[0]
    else:
        state["weight"], state["bias"] = (1 + 0.1 * _randn((n,), g)).to(dt), (0.1 * _randn((n,), g)).to(dt)
    if c["train"]:
        state["dy"] = _randn((b, s, n), g).to(dt)
    return state


def prepare(case: dict, seed: int) -> dict:
    state = _inputs(case, seed)
    if case["kind"] == "wgrad":  # the backward pass has the kept input, not the input
        x = state.pop("x")
        if own:
            from stagehand_amd.act8 import quantize_activation

            state["kept"] = quantize_activation(x)
        else:
            state["kept"] = _plain_quantize(x)
    elif case["kind"] == "norm" and case["train"]:
        for name in ("x", "weight", "bias"):
            state[name] = state[name].detach().requires_grad_()
    state["case"] = case
    return state


# ── one pass ─────────────────────────────────────────────────────────────────


def run(state: dict):
    kind = state["case"]["kind"]
    if own:
        return {"norm": _own_norm, "keep": _own_keep, "wgrad": _own_wgrad}[kind](state)
    with torch.no_grad():
        return {"norm": _plain_norm, "keep": _plain_keep, "wgrad": _plain_wgrad}[kind](state)


def _own_norm(s: dict):
    from stagehand_amd.layer_norm import layer_norm

    c = s["case"]
    y = layer_norm(s["x"], s["weight"], s["bias"], eps=EPS, modulate=c["modulate"], keep8=c["keep8"] and c["train"])
    if not c["train"]:
        return {"y": y}
    dx, dw, db = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])
    return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}


def _own_keep(s: dict):
    from stagehand_amd.act8 import quantize_activation

    return quantize_activation(s["x"]).dequantize()


def _own_wgrad(s: dict):
    from stagehand_amd.act8 import weight_grad_act8

    dw, db = weight_grad_act8(s["dy"], s["kept"], bias=s["case"]["bias"])
    return {"dweight": dw, "dbias": db} if s["case"]["bias"] else {"dweight": dw}


def _plain_quantize(x: torch.Tensor):
    """(q as int8 groups of 32, the powers' exponents, the activation's width and type)."""
    cols = x.shape[-1]
    v = torch.nn.functional.pad(x.float(), (0, -cols % 32)).unflatten(-1, (-1, 32))
    # max |x| = 1.f * 2^E, and 127 * 2^k = 1.984375 * 2^(k + 6): k = E - 6, one more for 1.f > 1.984375
    bits = v.abs().amax(-1, keepdim=True).view(torch.int32)
    k = (((bits + 0x1FFFF) >> 23) - 133).clamp_min(-126)
    # both factors are powers of two within the range: the product is exact
    inverse = ((127 - k) << 23).view(torch.float32)
    most = torch.where(k == (10 if x.dtype == torch.float16 else 122), 63.0, 127.0)
    q = torch.minimum(torch.maximum(torch.round(v * inverse), -most), most)
    return q.to(torch.int8), k, cols, x.dtype


def _plain_dequantize(kept) -> torch.Tensor:
    """The kept values, in 32 bits."""
    q, k, cols, _ = kept
    return (q.float() * ((127 + k) << 23).view(torch.float32)).flatten(-2)[..., :cols]


def _plain_keep(s: dict):
    kept = _plain_quantize(s["x"])
    return _plain_dequantize(kept).to(kept[3])


def _plain_wgrad(s: dict):
    dy = s["dy"].float()
    out = {"dweight": (dy.t() @ _plain_dequantize(s["kept"])).to(s["dy"].dtype)}
    if s["case"]["bias"]:
        out["dbias"] = dy.sum(0).to(s["dy"].dtype)
    return out


def _plain_norm(s: dict):
    c, dt = s["case"], s["x"].dtype
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    if c["modulate"]:
        w = 1 + w
    mean = x.mean(-1, keepdim=True)
    d = x - mean
    r = torch.rsqrt((d * d).mean(-1, keepdim=True) + EPS)
    n = d * r
    out = {"y": (n * w + b).to(dt)}
    if c["train"]:
        if c["keep8"]:
            n = (_plain_dequantize(_plain_quantize(s["x"])) - mean) * r
        dy = s["dy"].float()
        g = dy * w
        out["dx"] = (r * (g - g.mean(-1, keepdim=True) - n * (g * n).mean(-1, keepdim=True))).to(dt)
        dims = (1,) if c["modulate"] else (0, 1)
        out["dweight"] = (dy * n).sum(dims).view(s["weight"].shape).to(dt)
        out["dbias"] = dy.sum(dims).view(s["bias"].shape).to(dt)
    return out


# ── what a pass cannot do without, and its results in 64 bits ────────────────


def work(case: dict) -> dict:
    c = case
    e = 4 if c["dtype"] == "f32" else 2
    kept = 1 + 1 / 32
    if c["kind"] == "keep":
        values = c["tokens"] * c["cols"]
        return {"bytes": (2 * e + 2 * kept) * values, "flops": 4.0 * values}
    if c["kind"] == "wgrad":
        t, o, i = c["tokens"], c["out"], c["inp"]
        return {"bytes": t * o * e + kept * t * i + o * i * e + c["bias"] * o * e, "flops": 2.0 * t * o * i}
    values = c["batch"] * c["seq"] * c["cols"]
    params = 2 * e * c["cols"] * (c["batch"] if c["modulate"] else 1)
    if not c["train"]:
        return {"bytes": 2 * e * values + params, "flops": 7.0 * values}
    # forward: x in, y out; backward: x (or what is kept of it, which the forward writes) and dy in, dx out
    return {"bytes": ((4 * e + 2 * kept) if c["keep8"] else 5 * e) * values + 3 * params, "flops": 20.0 * values}


def _exact_kept(x: torch.Tensor) -> torch.Tensor:
    """What an activation is when it has been kept in 8 bits."""
    cols, top = x.shape[-1], torch.finfo(x.dtype).max
    v = x.double()
    if cols % 32:
        v = torch.cat((v, v.new_zeros(*v.shape[:-1], 32 - cols % 32)), -1)
    v = v.reshape(*v.shape[:-1], -1, 32)
    m, e = torch.frexp(v.abs().amax(-1))  # m * 2^e is at most 127 * 2^(e - 7) if m is at most 127/128
    e = torch.where(m <= 127 / 128, e - 7, e - 6).clamp_min(-126)
    step = ((e.long() + 1023) << 52).view(torch.float64)[..., None]  # 2^e as a double
    kept = torch.round(v / step) * step
    kept = torch.where(kept.abs() > top, kept - step * kept.sign(), kept)
    return kept.reshape(*x.shape[:-1], -1)[..., :cols]


def exact(case: dict, seed: int):
    c, s = case, _inputs(case, seed)
    if c["kind"] == "keep":
        return _exact_kept(s["x"])
    if c["kind"] == "wgrad":
        kept, dy = _exact_kept(s["x"]), s["dy"].double()
        out = {"dweight": dy.t().contiguous() @ kept}
        if c["bias"]:
            out["dbias"] = dy.sum(0)
        return out
    x, w, b = s["x"].double(), s["weight"].double(), s["bias"].double()
    gain = w + 1 if c["modulate"] else w
    var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
    std = (var + EPS).sqrt()
    out = {"y": (x - mean) / std * gain + b}
    if c["train"]:
        n = ((_exact_kept(s["x"]) if c["keep8"] else x) - mean) / std
        del x
        dy = s["dy"].double()
        share = tuple(range(1 if c["modulate"] else 0, 2))
        out["dweight"] = (dy * n).sum(share).reshape(w.shape)
        out["dbias"] = dy.sum(share).reshape(b.shape)
        g = dy.mul_(gain)
        out["dx"] = (g - g.mean(-1, keepdim=True) - n * (g * n).mean(-1, keepdim=True)) / std
    return out
