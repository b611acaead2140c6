"""The training-step operators this package is timed on: group norm with an activation on channels-last maps, the gated
feed-forward product, and the global gradient norm with clipping, at the sizes a program meets that trains or runs gated
refiner blocks, from one row to the largest maps.

A case names a ``kind`` and its sizes; ``train`` adds the backward pass. With ``own`` false, :func:`run` computes the
operator from elementary torch operations in 32 bits, rounded once at the end; with ``own`` true it calls the package's
entry points. :func:`exact` is the same from the definitions in 64 bits.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-5
CLIP_EPS = 1e-6  # beside the norm in the clip's quotient


def listed() -> list[dict]:
    return [
        # the smallest map: 1/32 of a 1024 x 1024 image; launch latency counts
        dict(name="norm_64_32x32", kind="norm", b=1, h=32, w=32, c=64, groups=8, act="silu", dtype="bf16", param="bf16",
             train=False),
        # two 200 x 200 maps in front of a quantized layer
        dict(name="norm_128_200x200", kind="norm", b=2, h=200, w=200, c=128, groups=32, act="gelu", dtype="bf16",
             param="bf16", train=False),
        # a training step at the finest scale: 64 channels on two 400 x 400 maps, FP32 parameters
        dict(name="norm_train_64_400x400", kind="norm", b=2, h=400, w=400, c=64, groups=8, act="gelu", dtype="bf16",
             param="fp32", train=True),
        # FP32 training on odd maps with a channel count that is no multiple of 16
        dict(name="norm_train_196_75x101", kind="norm", b=3, h=75, w=101, c=196, groups=14, act="silu", dtype="fp32",
             param="fp32", train=True),
        # one row (a pooled descriptor): the weights are the traffic
        dict(name="gated_512_one_row", kind="gated", rows=1, k=512, hidden=2048, act="silu", dtype="bf16", bias="none",
             train=False),
        # the feed-forward of a 512-channel block on two 100 x 100 maps
        dict(name="gated_512_20000", kind="gated", rows=20000, k=512, hidden=2048, act="gelu", dtype="bf16", bias="same",
             train=False),
        # a training step at the finest scale: few channels, 320000 pixels
        dict(name="gated_train_64_320000", kind="gated", rows=320000, k=64, hidden=256, act="silu", dtype="bf16",
             bias="same", train=True),
        # FP16 training with sizes that are no multiples of anything (a 112 x 150 map, 8/3 of 196 hidden channels)
        dict(name="gated_train_196_16800", kind="gated", rows=16800, k=196, hidden=523, act="gelu_tanh", dtype="fp16",
             bias="fp32", train=True),
        # a wide feed-forward's training step: large matrix products
        dict(name="gated_train_1024_16384", kind="gated", rows=16384, k=1024, hidden=4096, act="silu", dtype="bf16",
             bias="none", train=True),
        # the gradients of one 64-channel refiner block: ten tensors
        dict(name="clip_block_64", kind="clip", sizes="refiner", channels=64, blocks=1, dtype="fp32", out="fp32",
             norm=2.0, max_norm=1.0),
        # the gradients of the refiner stack's four scales, eight blocks each: 320 tensors
        dict(name="clip_stack", kind="clip", sizes="refiner", channels=0, blocks=8, dtype="fp32", out="fp32", norm=2.0,
             max_norm=1.0),
        # a large model's BF16 gradients, clipped into the FP32 ones that its optimizer reads
        dict(name="clip_wide_bf16", kind="clip", sizes="random", tensors=132, elements=200_000_000, dtype="bf16",
             out="fp32", norm=2.0, max_norm=0.5),
    ]


CHANNELS = (32, 64, 96, 128, 192, 196, 256, 320, 384, 512)
# a backward pass through a ReLU jumps where the sum behind it is zero up to its rounding: forward passes only
SMOOTH = ("none", "silu", "gelu", "gelu_tanh")
MOST_NORM = 2 * 400 * 400 * 64  # elements of a drawn map
MOST_GATED = 12 * 16384 * 1024 * 4096.0  # flops of a drawn feed-forward
MOST_CLIP = 150_000_000  # elements


def _log_uniform(rng, lo: float, hi: float) -> float:
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def draw(rng) -> dict:
    kind = rng.choice(("norm", "norm", "gated", "gated", "clip"))
    if kind == "norm":
        c = rng.choice(CHANNELS)
        b = rng.choice((1, 1, 2, 2, 3))
        pixels = _log_uniform(rng, 256, MOST_NORM / c) / b
        aspect = _log_uniform(rng, 0.5, 2.0)
        h, w = max(1, int(math.sqrt(pixels * aspect))), max(1, int(math.sqrt(pixels / aspect)))
        dtype, train = rng.choice(("bf16", "bf16", "fp16", "fp32")), rng.random() < 0.6
        return dict(kind=kind, b=b, h=h, w=w, c=c, groups=rng.choice([g for g in (1, 4, 8, 14, 16, 32) if c % g == 0]),
                    act=rng.choice(SMOOTH if train else SMOOTH + ("relu",)), dtype=dtype, param=rng.choice((dtype, "fp32")),
                    train=train)
    if kind == "gated":
        while True:
            k = rng.choice(CHANNELS + (640, 1000, 1024))
            hidden = rng.choice((2 * k, 4 * k, 8 * k // 3))
            rows = round(_log_uniform(rng, 1, 320000))
            train = rows > 16 and rng.random() < 0.6
            case = dict(kind=kind, rows=rows, k=k, hidden=hidden,
                        act=rng.choice(SMOOTH[1:] if train else SMOOTH[1:] + ("relu",)),
                        dtype=rng.choice(("bf16", "bf16", "fp16")), bias=rng.choice(("none", "same", "fp32")), train=train)
            if work(case)["flops"] <= MOST_GATED and work(case)["bytes"] <= 1.2e9 and 3072 not in (rows, hidden):
                return case
    dtype = rng.choice(("fp32", "bf16", "fp16"))
    case = dict(kind=kind, sizes="random", tensors=round(_log_uniform(rng, 1, 400)),
                elements=round(_log_uniform(rng, 20000, MOST_CLIP)), dtype=dtype, out=rng.choice((dtype, "fp32")),
                norm=rng.choice((2.0, 2.0, math.inf)), max_norm=rng.choice((0.1, 1.0, 1e4)))
    return case


# -- inputs ----------------------------------------------------------------------------------------------------------


def _randn(g, *shape) -> torch.Tensor:
    return torch.randn(*shape, generator=g, device=DEV)


def _spread(g, n: int) -> torch.Tensor:
    """Per-channel factors between 0.3 and 3, as measured activations have."""
    return torch.exp(torch.empty(n, device=DEV).uniform_(math.log(0.3), math.log(3.0), generator=g))


def _tensor_sizes(c: dict) -> list[int]:
    """Element counts of the gradients of a clip case."""
    if c["sizes"] == "refiner":  # a refiner block's depthwise weight, five vectors, two matrices and their biases
        sizes = []
        for ch in ([c["channels"]] if c["channels"] else [512, 256, 128, 64]):
            sizes += [25 * ch, ch, ch, ch, ch, ch, 4 * ch * ch, 4 * ch, 4 * ch * ch, ch] * c["blocks"]
        return sizes
    rng = random.Random(c["tensors"] * 1_000_003 + c["elements"])
    share = [math.exp(rng.uniform(0.0, 8.0)) for _ in range(c["tensors"])]
    return [max(1, int(c["elements"] * s / sum(share))) for s in share]


def prepare(case: dict, seed: int) -> dict:
    c, g = case, torch.Generator(device=DEV).manual_seed(seed)
    if c["kind"] == "clip":
        sizes = _tensor_sizes(c)
        bucket = torch.empty(sum(sizes), dtype=DTYPES[c["dtype"]], device=DEV)  # gradients lie packed, as views
        grads = list(bucket.split(sizes))
        factors = torch.exp(torch.empty(len(sizes)).uniform_(-6.0, 0.0, generator=torch.Generator().manual_seed(seed)))
        for grad, factor in zip(grads, factors.tolist()):
            grad.normal_(0.0, factor, generator=g)
        out = torch.empty(bucket.numel(), dtype=DTYPES[c["out"]], device=DEV)
        return dict(case=c, bucket=bucket, grads=grads, out_bucket=out, out=list(out.split(sizes)))
    dtype = DTYPES[c["dtype"]]
    if c["kind"] == "norm":
        shape, p = (c["b"], c["h"], c["w"], c["c"]), DTYPES[c["param"]]
        x = (_randn(g, *shape) * _spread(g, c["c"]) + _randn(g, c["c"])).to(dtype)
        state = dict(case=c, x=x, weight=(1 + 0.2 * _randn(g, c["c"])).to(p), bias=(0.2 * _randn(g, c["c"])).to(p))
        inputs, out_shape = ("x", "weight", "bias"), shape
    else:
        m, k, h = c["rows"], c["k"], c["hidden"]
        state = dict(case=c, x=(_randn(g, m, k) * _spread(g, k)).to(dtype))
        state |= dict(w_gate=(_randn(g, h, k) * k ** -0.5).to(dtype), w_up=(_randn(g, h, k) * k ** -0.5).to(dtype),
                      b_gate=None, b_up=None)
        if c["bias"] != "none":
            b = dtype if c["bias"] == "same" else torch.float32
            state |= dict(b_gate=(0.2 * _randn(g, h)).to(b), b_up=(0.2 * _randn(g, h)).to(b))
        inputs, out_shape = ("x", "w_gate", "w_up", "b_gate", "b_up"), (m, h)
    if c["train"]:
        state["d_out"] = (_randn(g, *out_shape) * 0.1).to(dtype)
        state["wanted"] = [state[n].requires_grad_() for n in inputs if state[n] is not None]
    return state


# -- one pass --------------------------------------------------------------------------------------------------------


def run(state: dict):
    c = state["case"]
    if not own:
        with torch.no_grad():
            return {"norm": _plain_norm, "gated": _plain_gated, "clip": _plain_clip}[c["kind"]](c, state)
    from flashim_amd import ops

    if c["kind"] == "clip":
        total = ops.clip_grad_norm_(state["grads"], c["max_norm"], norm_type=c["norm"], out=state["out"])
        return [total, state["out_bucket"]]
    if c["kind"] == "norm":
        out = ops.group_norm_act(state["x"], c["groups"], state["weight"], state["bias"], eps=EPS, activation=c["act"])
    else:
        out = ops.gated_linear(state["x"], state["w_gate"], state["w_up"], state["b_gate"], state["b_up"],
                               activation=c["act"])
    if not c["train"]:
        return [out]
    return [out.detach(), *torch.autograd.grad(out, state["wanted"], state["d_out"])]


def _activation(z: torch.Tensor, act: str) -> tuple[torch.Tensor, torch.Tensor]:
    """act(z) and act'(z)."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return z * (z > 0), (z > 0).to(z.dtype)
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    a, b = math.sqrt(2 / math.pi), 0.044715  # gelu_tanh
    t = torch.tanh(a * (z + b * z * z * z))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * a * (1 + 3 * b * z * z)


def _plain_norm(c: dict, s: dict):
    groups, d = c["groups"], c["c"] // c["groups"]
    x = s["x"].float().reshape(c["b"], -1, groups, d)
    weight, bias = s["weight"].float().reshape(groups, d), s["bias"].float().reshape(groups, d)
    centred = x - x.mean(dim=(1, 3), keepdim=True)
    rstd = (centred.square().mean(dim=(1, 3), keepdim=True) + EPS).rsqrt()
    xhat = centred * rstd
    y, slope = _activation(xhat * weight + bias, c["act"])
    y = y.to(s["x"].dtype).reshape(s["x"].shape)
    if not c["train"]:
        return [y]
    dz = s["d_out"].float().reshape(xhat.shape) * slope
    d_weight, d_bias = (dz * xhat).sum(dim=(0, 1)), dz.sum(dim=(0, 1))
    dz = dz * weight
    dx = rstd * (dz - dz.mean(dim=(1, 3), keepdim=True) - xhat * (dz * xhat).mean(dim=(1, 3), keepdim=True))
    return [y, dx.to(s["x"].dtype).reshape(s["x"].shape), d_weight.reshape(-1).to(s["weight"].dtype),
            d_bias.reshape(-1).to(s["bias"].dtype)]


def _plain_gated(c: dict, s: dict):
    x, wg, wu = s["x"].float(), s["w_gate"].float(), s["w_up"].float()
    gate, up = x @ wg.t(), x @ wu.t()
    if s["b_gate"] is not None:
        gate, up = gate + s["b_gate"].float(), up + s["b_up"].float()
    a, slope = _activation(gate, c["act"])
    out = (a * up).to(s["x"].dtype)
    if not c["train"]:
        return [out]
    d_out = s["d_out"].float()
    d_gate, d_up = d_out * up * slope, d_out * a
    grads = [d_gate @ wg + d_up @ wu, d_gate.t() @ x, d_up.t() @ x]
    if s["b_gate"] is not None:
        grads += [d_gate.sum(dim=0), d_up.sum(dim=0)]
    return [out, *(g.to(w.dtype) for g, w in zip(grads, s["wanted"]))]


def _plain_clip(c: dict, s: dict):
    x = s["bucket"].float()  # all gradients at once, as they lie packed
    total = x.square().sum().sqrt() if c["norm"] == 2.0 else x.abs().max()
    scale = (c["max_norm"] / (total + CLIP_EPS)).clamp(max=1.0)
    s["out_bucket"].copy_(x * scale)
    return [total, s["out_bucket"]]


# -- what a pass cannot do without -----------------------------------------------------------------------------------

SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def work(case: dict) -> dict:
    c = case
    if c["kind"] == "clip":
        n = sum(_tensor_sizes(c))
        return {"bytes": n * (SIZE[c["dtype"]] + SIZE[c["out"]]), "flops": 3 * n}
    if c["kind"] == "norm":  # x in and y out; the backward pass: d_out in and dx out
        n = c["b"] * c["h"] * c["w"] * c["c"]
        return {"bytes": n * SIZE[c["dtype"]] * (4 if c["train"] else 2), "flops": n * (30 if c["train"] else 12)}
    m, k, h = c["rows"], c["k"], c["hidden"]
    once = m * k + 2 * h * k + m * h
    return {"bytes": SIZE[c["dtype"]] * once * (2 if c["train"] else 1), "flops": 4.0 * m * k * h * (3 if c["train"] else 1)}


# -- the same in 64 bits ---------------------------------------------------------------------------------------------


def _phi64(z: torch.Tensor, act: str) -> torch.Tensor:
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * torch.special.erfc(-z / math.sqrt(2.0))
    if act == "gelu_tanh":
        return z / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z


def exact(case: dict, seed: int):
    c, s = case, prepare(case, seed)
    if c["kind"] == "clip":
        parts = [g.double() for g in s["grads"]]
        if c["norm"] == 2.0:
            total = torch.stack([p.norm() for p in parts]).norm()
        else:
            total = torch.stack([p.abs().amax() for p in parts]).amax()
        return [total, torch.cat(parts) * min(1.0, c["max_norm"] / (total.item() + CLIP_EPS))]
    names = [n for n in ("x", "weight", "bias", "w_gate", "w_up", "b_gate", "b_up") if s.get(n) is not None]
    v = {n: s[n].detach().double().requires_grad_(c["train"]) for n in names}
    if c["kind"] == "norm":
        rows = v["x"].reshape(c["b"], -1, c["groups"], c["c"] // c["groups"]).transpose(1, 2).flatten(2)
        var, mean = torch.var_mean(rows, dim=-1, unbiased=False, keepdim=True)
        xhat = ((rows - mean) / (var + EPS).sqrt()).unflatten(2, (-1, c["c"] // c["groups"])).transpose(1, 2)
        out = _phi64(xhat.reshape(v["x"].shape) * v["weight"] + v["bias"], c["act"])
    else:
        gate, up = v["x"] @ v["w_gate"].t(), v["x"] @ v["w_up"].t()
        if "b_gate" in v:
            gate, up = gate + v["b_gate"], up + v["b_up"]
        out = _phi64(gate, c["act"]) * up
    if not c["train"]:
        return [out]
    return [out.detach(), *torch.autograd.grad(out, [v[n] for n in names], s["d_out"].double())]
