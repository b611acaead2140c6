"""The operators this package is timed on for training and adapting gated blocks: orthogonalized updates by Newton-Schulz
products, the optimizer step made of them, and low-rank adapters of many requests beside a shared projection, at the sizes a
program meets that trains gated refiner blocks or serves one of them with adapters, from one row and one small matrix to the
largest maps and matrices.

A case names a ``kind`` and its sizes; ``train`` adds the backward pass. With ``own`` false, :func:`run` computes the
operator from elementary torch operations in 32 bits (norms of whole matrices in 64), rounded once at the end; with ``own``
true it calls the package's entry points. :func:`exact` is the same from the definitions in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
EPS = 1e-7  # beside the norm
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.1


def listed() -> list[dict]:
    return [
        # one matrix of a 64-channel block: latency counts
        dict(name="ortho_64x256", kind="ortho", batch=1, rows=64, cols=256, dtype="bf16"),
        # the first factors of 64 adapters of rank 16, trained in 32 bits
        dict(name="ortho_64_of_16x512", kind="ortho", batch=64, rows=16, cols=512, dtype="fp32"),
        # an odd, tall matrix: 196 channels, 8/3 of them inside
        dict(name="ortho_523x196", kind="ortho", batch=1, rows=523, cols=196, dtype="fp16"),
        # a wide block's projection
        dict(name="ortho_1024x4096", kind="ortho", batch=1, rows=1024, cols=4096, dtype="bf16"),
        # the optimizer step of one 64-channel gated block: gate, up and down matrices
        dict(name="muon_block_64", kind="muon", channels=64, hidden=256, blocks=1, param="bf16", grad="bf16"),
        # that of a refiner stack's four scales (512, 256, 128 and 64 channels), eight blocks each: 96 matrices
        dict(name="muon_stack", kind="muon", channels=0, hidden=0, blocks=8, param="fp32", grad="fp32"),
        # that of a wide block: BF16 gradients, FP32 parameters
        dict(name="muon_wide", kind="muon", channels=1024, hidden=4096, blocks=1, param="fp32", grad="bf16"),
        # one request of one row (a pooled descriptor)
        dict(name="adapt_one_row", kind="adapt", rows=1, images=1, k=512, n=2048, rank=8, adapters=4, dtype="bf16",
             index="image", train=False),
        # 64 requests of one row each, each with an adapter of its own: the adapters are the traffic
        dict(name="adapt_64_requests", kind="adapt", rows=64, images=64, k=1024, n=4096, rank=16, adapters=64,
             dtype="bf16", index="image", train=False),
        # four 100 x 100 maps beside a wide block's first projection
        dict(name="adapt_4_maps", kind="adapt", rows=40000, images=4, k=512, n=2048, rank=16, adapters=8, dtype="bf16",
             index="image", train=False),
        # a training step at the finest scale: two 400 x 400 maps
        dict(name="adapt_train_64_320000", kind="adapt", rows=320000, images=2, k=64, n=256, rank=8, adapters=2,
             dtype="bf16", index="image", train=True),
        # a training step over requests of uneven length, some without an adapter, at odd widths
        dict(name="adapt_train_ragged", kind="adapt", rows=16800, images=1, k=196, n=523, rank=12, adapters=6,
             dtype="fp16", index="row", train=True),
    ]


CHANNELS = (32, 64, 96, 128, 192, 196, 256, 320, 384, 512)
MOST_FLOPS = 3 * STEPS * (3.0 * 1024**2 * 4096 + 1024.0**3)  # of a drawn orthogonalization or step
MOST_BYTES = 5e8  # of a drawn adapter call


def _log_uniform(rng, lo: float, hi: float) -> float:
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def draw(rng) -> dict:
    kind = rng.choice(("ortho", "ortho", "muon", "adapt", "adapt", "adapt"))
    if kind == "ortho":
        while True:
            case = dict(kind=kind, batch=rng.choice((1, 1, 1, 2, 8, round(_log_uniform(rng, 1, 64)))),
                        rows=round(_log_uniform(rng, 4, 4096)), cols=round(_log_uniform(rng, 4, 4096)),
                        dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")))
            if work(case)["flops"] <= MOST_FLOPS and case["batch"] * case["rows"] * case["cols"] <= 2**24:
                return case
    if kind == "muon":
        channels = rng.choice(CHANNELS)
        param = rng.choice(("bf16", "fp16", "fp32"))
        return dict(kind=kind, channels=channels, hidden=rng.choice((2 * channels, 4 * channels, 8 * channels // 3)),
                    blocks=rng.choice((1, 2, 3, 5, 8)), param=param, grad=rng.choice((param, "bf16", "fp32")))
    while True:
        k, n = rng.choice(CHANNELS + (523, 1024)), rng.choice(CHANNELS + (523, 1024, 2048))
        index = rng.choice(("image", "row"))
        rows = round(_log_uniform(rng, 1, 320000 if index == "image" else 30000))
        images = rng.choice((1, 2, 3, 8, 64))
        case = dict(kind=kind, rows=-(-rows // images) * images, images=images, k=k, n=n,
                    rank=rng.choice((1, 4, 8, 12, 16, 32, 64)), adapters=rng.choice((1, 2, 6, 16, 64)),
                    dtype=rng.choice(("bf16", "bf16", "fp16")), index=index, train=rows > 16 and rng.random() < 0.5)
        per_row = case["rank"] * max(k, n) * 4 * (case["rows"] if index == "row" else images)
        if work(case)["bytes"] <= MOST_BYTES and per_row <= 2e9:  # (the plain form's adapters, gathered)
            return case


# -- inputs ----------------------------------------------------------------------------------------------------------


def _randn(g, *shape) -> torch.Tensor:
    return torch.randn(*shape, generator=g, device=DEV)


def _gradient(g, count: int, rows: int, cols: int) -> torch.Tensor:
    """Matrices as gradients are: a few strong directions, each e^-0.5 of the one before, over a floor of noise."""
    few = min(8, rows, cols)
    decay = torch.exp(-0.5 * torch.arange(few, device=DEV))
    return (torch.matmul(_randn(g, count, rows, few) * decay, _randn(g, count, few, cols))
            + 0.05 * _randn(g, count, rows, cols)) * 1e-3


def _matrices(c: dict) -> list[tuple[int, int, int]]:
    """(count, rows, cols) of a step's matrices as they lie behind each other: gate and up, then down, scale by scale."""
    groups = []
    for channels in ([c["channels"]] if c["channels"] else [512, 256, 128, 64]):
        hidden = c["hidden"] or 4 * channels
        groups += [(2 * c["blocks"], hidden, channels), (c["blocks"], channels, hidden)]
    return groups


def _stacks(bucket: torch.Tensor, groups: list[tuple[int, int, int]]) -> list[torch.Tensor]:
    parts = bucket.split([n * r * k for n, r, k in groups])
    return [p.view(shape) for p, shape in zip(parts, groups)]


def _index(c: dict, g) -> torch.Tensor:
    """An adapter for each image, or for each row in runs of uneven length of which one in eight has none."""
    if c["index"] == "image":
        if c["adapters"] >= c["images"]:
            return torch.randperm(c["adapters"], generator=g, device=DEV)[:c["images"]]
        return torch.randint(0, c["adapters"], (c["images"],), generator=g, device=DEV)
    runs = max(1, min(c["rows"], 4 * c["adapters"]))
    ends = torch.sort(torch.randint(0, c["rows"], (runs,), generator=g, device=DEV)).values
    which = torch.randint(0, c["adapters"], (runs + 1,), generator=g, device=DEV)
    which = torch.where(torch.rand(runs + 1, generator=g, device=DEV) < 0.125, torch.full_like(which, -1), which)
    return which[torch.searchsorted(ends, torch.arange(c["rows"], device=DEV))]


def prepare(case: dict, seed: int) -> dict:
    c, g = case, torch.Generator(device=DEV).manual_seed(seed)
    if c["kind"] == "ortho":
        x = _gradient(g, c["batch"], c["rows"], c["cols"]).to(DTYPES[c["dtype"]])
        return dict(case=c, g=x if c["batch"] > 1 else x[0])
    if c["kind"] == "muon":
        groups = _matrices(c)
        total = sum(n * r * k for n, r, k in groups)
        state = dict(case=c, params=torch.empty(total, dtype=DTYPES[c["param"]], device=DEV),
                     grads=torch.empty(total, dtype=DTYPES[c["grad"]], device=DEV),
                     momenta=torch.empty(total, device=DEV))
        stacks = {name: _stacks(state[name], groups) for name in ("params", "grads", "momenta")}
        for i, (n, rows, cols) in enumerate(groups):
            stacks["params"][i].copy_(_randn(g, n, rows, cols) * cols ** -0.5)
            stacks["grads"][i].copy_(_gradient(g, n, rows, cols))
            stacks["momenta"][i].copy_(5 * _gradient(g, n, rows, cols))
        state["stacks"] = stacks
        state["lists"] = {name: [m for stack in s for m in stack.unbind()] for name, s in stacks.items()}
        return state
    dtype = DTYPES[c["dtype"]]
    lead = (c["images"], c["rows"] // c["images"]) if c["index"] == "image" else (c["rows"],)
    spread = torch.exp(torch.empty(c["k"], device=DEV).uniform_(math.log(0.3), math.log(3.0), generator=g))
    state = dict(case=c, x=(_randn(g, *lead, c["k"]) * spread).to(dtype), base=_randn(g, *lead, c["n"]).to(dtype),
                 a=(_randn(g, c["adapters"], c["rank"], c["k"]) * c["k"] ** -0.5).to(dtype),
                 b=(_randn(g, c["adapters"], c["n"], c["rank"]) * 0.3 * c["rank"] ** -0.5).to(dtype),
                 scale=torch.exp(torch.empty(c["adapters"], device=DEV).uniform_(-0.7, 0.7, generator=g)),
                 index=_index(c, g))
    if c["train"]:
        state["d_out"] = (_randn(g, *lead, c["n"]) * 0.1).to(dtype)
        state["wanted"] = [state[n].requires_grad_() for n in ("x", "a", "b")]
    return state


# -- one pass --------------------------------------------------------------------------------------------------------


def run(state: dict):
    c = state["case"]
    if not own:
        with torch.no_grad():
            return {"ortho": _plain_ortho, "muon": _plain_muon, "adapt": _plain_adapt}[c["kind"]](c, state)
    from flashim_amd import ops

    if c["kind"] == "ortho":
        return [ops.orthogonalize(state["g"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)]
    if c["kind"] == "muon":
        lists = state["lists"]
        ops.muon_step_(lists["params"], lists["grads"], lists["momenta"], lr=LR, momentum=MOMENTUM, nesterov=True,
                       weight_decay=DECAY, steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)
        return [state["params"], state["momenta"]]
    out = ops.low_rank_adapters(state["base"], state["x"], state["a"], state["b"], state["index"], scale=state["scale"])
    if not c["train"]:
        return [out]
    return [out.detach(), *torch.autograd.grad(out, state["wanted"], state["d_out"])]


def _newton_schulz(u: torch.Tensor) -> torch.Tensor:
    """Of matrices [..., rows, cols] in 32 bits, their norms in 64."""
    norm = u.double().square().sum(dim=(-2, -1), keepdim=True).sqrt() + EPS
    x = (u.double() / norm).float()
    tall = x.shape[-2] > x.shape[-1]
    x = x.transpose(-2, -1).contiguous() if tall else x
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        gram = x @ x.transpose(-2, -1).contiguous()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.transpose(-2, -1) if tall else x


def _plain_ortho(c: dict, s: dict):
    return [_newton_schulz(s["g"].float()).to(s["g"].dtype).contiguous()]


def _plain_muon(c: dict, s: dict):
    for p, grad, m in zip(*(s["stacks"][n] for n in ("params", "grads", "momenta"))):  # stacks of one shape
        u = grad.float()
        m.mul_(MOMENTUM).add_(u)
        o = _newton_schulz(u + MOMENTUM * m)
        factor = LR * math.sqrt(max(1.0, p.shape[-2] / p.shape[-1]))
        p.copy_(p.float() * (1 - LR * DECAY) - factor * o)
    return [s["params"], s["momenta"]]


def _plain_adapt(c: dict, s: dict):
    entries = s["index"].numel()
    some = s["index"] >= 0
    which = s["index"].clamp(min=0)
    a, b = s["a"].float()[which], s["b"].float()[which]  # [entries, R, K], [entries, N, R]
    scale = torch.where(some, s["scale"][which], torch.zeros_like(s["scale"][which]))[:, None, None]
    x = s["x"].float().reshape(entries, -1, c["k"])
    h = torch.matmul(x, a.transpose(1, 2).contiguous()) * scale
    out = s["base"].float() + torch.matmul(h, b.transpose(1, 2).contiguous()).reshape(s["base"].shape)
    out = out.to(s["base"].dtype)
    if not c["train"]:
        return [out]
    d = s["d_out"].float().reshape(entries, -1, c["n"])
    t = torch.matmul(d, b) * scale
    dx = torch.matmul(t, a).reshape(s["x"].shape)
    da = torch.zeros_like(s["a"], dtype=torch.float32).index_add_(0, which, torch.matmul(t.transpose(1, 2).contiguous(), x))
    db = torch.zeros_like(s["b"], dtype=torch.float32).index_add_(0, which, torch.matmul(d.transpose(1, 2).contiguous(), h))
    return [out, dx.to(s["x"].dtype), da.to(s["a"].dtype), db.to(s["b"].dtype)]


# -- what a pass cannot do without -----------------------------------------------------------------------------------

SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def _schulz_flops(rows: int, cols: int) -> float:
    """Two symmetric products, half of each, and one whole one a step."""
    m, n = min(rows, cols), max(rows, cols)
    return STEPS * (3.0 * m * m * n + 1.0 * m**3)


def work(case: dict) -> dict:
    c = case
    if c["kind"] == "ortho":
        n = c["batch"] * c["rows"] * c["cols"]
        return {"bytes": 2 * n * SIZE[c["dtype"]], "flops": c["batch"] * _schulz_flops(c["rows"], c["cols"])}
    if c["kind"] == "muon":  # the gradient in, parameter and momentum in and out
        groups = _matrices(c)
        total = sum(n * r * k for n, r, k in groups)
        return {"bytes": total * (SIZE[c["grad"]] + 2 * SIZE[c["param"]] + 8),
                "flops": sum(n * _schulz_flops(r, k) for n, r, k in groups)}
    m, k, n, rank = c["rows"], c["k"], c["n"], c["rank"]
    used = min(c["adapters"], c["images"]) if c["index"] == "image" else min(c["adapters"], m)
    weights = used * rank * (k + n)
    elements, flops = m * (k + 2 * n) + weights, 2.0 * m * rank * (k + n)
    if c["train"]:  # x and d_out in, dx and the adapters' gradients out
        elements, flops = elements + m * (2 * k + n) + 2 * weights, 3 * flops
    return {"bytes": elements * SIZE[c["dtype"]], "flops": flops}


# -- the same in 64 bits ---------------------------------------------------------------------------------------------


def _schulz64(u: torch.Tensor) -> torch.Tensor:
    """Of one matrix, from the left or the right, whichever makes the smaller products."""
    a, b, c = COEFFICIENTS
    x = u / (torch.linalg.vector_norm(u) + EPS)
    for _ in range(STEPS):
        if x.shape[0] <= x.shape[1]:
            gram = torch.mm(x, x.t())
            x = a * x + torch.mm(b * gram + c * torch.mm(gram, gram), x)
        else:
            gram = torch.mm(x.t(), x)
            x = a * x + torch.mm(x, b * gram + c * torch.mm(gram, gram))
    return x


def exact(case: dict, seed: int):
    c, s = case, prepare(case, seed)
    if c["kind"] == "ortho":
        g = s["g"].double()
        return [torch.stack([_schulz64(m) for m in g.reshape(-1, *g.shape[-2:])]).reshape(g.shape)]
    if c["kind"] == "muon":
        params, momenta = [], []
        for p, grad, m in zip(*(s["lists"][n] for n in ("params", "grads", "momenta"))):
            grad, m = grad.double(), m.double()
            m = MOMENTUM * m + grad
            rows, cols = p.shape
            step = LR * max(1.0, rows / cols) ** 0.5 * _schulz64(grad + MOMENTUM * m)
            params.append((p.double() - LR * DECAY * p.double() - step).reshape(-1))
            momenta.append(m.reshape(-1))
        return [torch.cat(params), torch.cat(momenta)]
    v = {n: s[n].detach().double().requires_grad_(c["train"]) for n in ("x", "a", "b")}
    rows_index = s["index"].repeat_interleave(c["rows"] // s["index"].numel())
    x, out = v["x"].reshape(-1, c["k"]), s["base"].double().reshape(-1, c["n"])
    for j in range(c["adapters"]):
        at = (rows_index == j).nonzero().squeeze(1)
        out = out.index_add(0, at, s["scale"][j].double() * torch.mm(torch.mm(x[at], v["a"][j].t()), v["b"][j].t()))
    out = out.reshape(s["base"].shape)
    if not c["train"]:
        return [out]
    return [out.detach(), *torch.autograd.grad(out, [v[n] for n in ("x", "a", "b")], s["d_out"].double())]
