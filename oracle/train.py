"""The training-step operators from their definitions in float64 on the CPU, gradients by their formulas. Each gradient
comes with the sum of the magnitudes that make it up (``terms``) where a test needs a bound on its rounding."""

from __future__ import annotations

import math

import torch
from torch import Tensor


def activation(z: Tensor, act: str) -> tuple[Tensor, Tensor]:
    """``act(z)`` and its derivative, float64."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return torch.maximum(z, torch.zeros_like(z)), (~(z <= 0)).to(z.dtype)  # (1 at NaN, as autograd has it)
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    if act == "gelu":
        cdf = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        a, b = math.sqrt(2 / math.pi), 0.044715
        t = torch.tanh(a * (z + b * z**3))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * a * (1 + 3 * b * z * z)
    raise ValueError(act)


def _grouped(x: Tensor, groups: int) -> Tensor:
    return x.reshape(x.shape[0], -1, groups, x.shape[-1] // groups)


def normalized(x: Tensor, groups: int, eps: float) -> tuple[Tensor, Tensor, Tensor]:
    """``(xhat, mean, rstd)`` of ``[B, ..., C]``; ``xhat`` in ``x``'s shape, the others ``[B, 1, groups, 1]``."""
    v = _grouped(x.double(), groups)
    mean = v.mean(dim=(1, 3), keepdim=True)
    rstd = 1 / torch.sqrt(((v - mean) ** 2).mean(dim=(1, 3), keepdim=True) + eps)
    return ((v - mean) * rstd).reshape(x.shape), mean, rstd


def group_norm_act(x: Tensor, groups: int, weight: Tensor | None, bias: Tensor | None, eps: float, act: str) -> Tensor:
    z = normalized(x, groups, eps)[0]
    z = z if weight is None else z * weight.double()
    return activation(z if bias is None else z + bias.double(), act)[0]


def group_norm_act_gradients(d_out: Tensor, x: Tensor, groups: int, weight: Tensor | None, bias: Tensor | None,
                             eps: float, act: str) -> dict[str, Tensor]:
    c = x.shape[-1]
    xhat, _, rstd = normalized(x, groups, eps)
    w = torch.ones(c, dtype=torch.float64) if weight is None else weight.double()
    z = xhat * w if bias is None else xhat * w + bias.double()
    dz = d_out.double() * activation(z, act)[1]
    rows, hat = dz.reshape(-1, c), xhat.reshape(-1, c)
    g, gh = _grouped(dz * w, groups), _grouped(xhat, groups)
    s1, s2 = g.mean(dim=(1, 3), keepdim=True), (g * gh).mean(dim=(1, 3), keepdim=True)
    m1, m2 = g.abs().mean(dim=(1, 3), keepdim=True), (g * gh).abs().mean(dim=(1, 3), keepdim=True)
    return {
        "x": (rstd * (g - s1 - gh * s2)).reshape(x.shape),
        "weight": (rows * hat).sum(0), "bias": rows.sum(0),
        "x_terms": (rstd * (g.abs() + m1 + gh.abs() * m2)).reshape(x.shape),
        "weight_terms": (rows * hat).abs().sum(0), "bias_terms": rows.abs().sum(0),
    }


def _pre(x: Tensor, w: Tensor, b: Tensor | None) -> tuple[Tensor, Tensor]:
    """``x w^T + b`` of ``[M, K]`` and the sum of its terms' magnitudes."""
    v, t = x.double() @ w.double().t(), x.double().abs() @ w.double().abs().t()
    return (v, t) if b is None else (v + b.double(), t + b.double().abs())


def gated_linear(x, w_gate, w_up, b_gate, b_up, act: str) -> tuple[Tensor, Tensor]:
    """The output of ``x [M, K]``, and how far it moves where each pre-activation moves by its terms' magnitudes."""
    (g, tg), (u, tu) = _pre(x, w_gate, b_gate), _pre(x, w_up, b_up)
    a, slope = activation(g, act)
    return a * u, (slope.abs() + 0.2) * tg * u.abs() + a.abs() * tu


def gated_linear_gradients(d_out, x, w_gate, w_up, b_gate, b_up, act: str) -> dict[str, Tensor]:
    """Gradients; ``*_terms`` the sums of their terms' magnitudes, ``*_squares`` the roots of the sums of the terms'
    squares (what rounding each pre-activation's gradient independently scales with)."""
    g, u = _pre(x, w_gate, b_gate)[0], _pre(x, w_up, b_up)[0]
    a, slope = activation(g, act)
    d, x, wg, wu = d_out.double(), x.double(), w_gate.double(), w_up.double()
    dg, du = d * u * slope, d * a
    return {
        "x": dg @ wg + du @ wu, "w_gate": dg.t() @ x, "w_up": du.t() @ x, "b_gate": dg.sum(0), "b_up": du.sum(0),
        "x_terms": dg.abs() @ wg.abs() + du.abs() @ wu.abs(),
        "x_squares": ((dg**2) @ (wg**2) + (du**2) @ (wu**2)).sqrt(),
        "w_gate_terms": dg.abs().t() @ x.abs(), "w_gate_squares": ((dg**2).t() @ (x**2)).sqrt(),
        "w_up_terms": du.abs().t() @ x.abs(), "w_up_squares": ((du**2).t() @ (x**2)).sqrt(),
        "b_gate_terms": dg.abs().sum(0), "b_up_terms": du.abs().sum(0),
    }


def grad_norm(grads, norm_type: float = 2.0) -> Tensor:
    flat = torch.cat([g.double().reshape(-1) for g in grads])
    return flat.square().sum().sqrt() if norm_type == 2.0 else flat.abs().max()


def clip_scale(total: Tensor, max_norm: float) -> Tensor:
    return torch.clamp(max_norm / (total.double() + 1e-6), max=1.0)


NEWTON_SCHULZ = (3.4445, -4.7750, 2.0315)


def schulz_iterates(u: Tensor, steps: int = 5, coefficients=NEWTON_SCHULZ, eps: float = 1e-7) -> list[Tensor]:
    """``[X_0, ..., X_steps]`` of one matrix, by its definition from the left (``rows <= cols``) or the right."""
    a, b, c = coefficients
    u = u.double()
    xs = [u / (u.square().sum().sqrt() + eps)]
    for _ in range(steps):
        x = xs[-1]
        if x.shape[0] <= x.shape[1]:
            gram = x @ x.t()
            xs.append(a * x + (b * gram + c * gram @ gram) @ x)
        else:
            gram = x.t() @ x
            xs.append(a * x + x @ (b * gram + c * gram @ gram))
    return xs


def orthogonalize(u: Tensor, **kwargs) -> Tensor:
    """Of ``[..., rows, cols]``."""
    flat = u.reshape(-1, *u.shape[-2:])
    return torch.stack([schulz_iterates(m, **kwargs)[-1] for m in flat]).reshape(u.shape)


def schulz_bound(u: Tensor, steps: int = 5, coefficients=NEWTON_SCHULZ, eps: float = 1e-7) -> float:
    """How far (Frobenius) an iteration of 22-bit operands and FP32 sums may end from one matrix's exact result.

    Step k's rounding is an error of at most e_k |X_k|: each product's operands are off by 2^-23, the dropped product of the
    low halves by 2^-24, and a sum of K terms, rounded K / 16 times or more at 2^-24 each, by 4 sqrt(K) 2^-24 (independent
    roundings); three products a step, whose factors a, b |A| and c |A|^2 multiply them by at most |a| + 2 |b| + 2 |c|. Besides, a low half
    below FP16's normal numbers, 2^-14, may count as zero: with the scales of 2^13 and more that go with singular values of at
    most 2, 2^-27 of each entry. Later
    steps multiply an error by at most the largest slope of the polynomial that is left (of an odd matrix function), between 0
    and the largest singular value."""
    a, b, c = coefficients
    m, n = sorted(u.shape[-2:])
    e = (2.0**-21 + 4 * math.sqrt(n) * 2.0**-24) * (abs(a) + 2 * abs(b) + 2 * abs(c))
    xs = schulz_iterates(u, steps, coefficients, eps)
    total = 0.0
    for k, x in enumerate(xs[:-1]):
        top = torch.linalg.matrix_norm(x, ord=2).item() * 1.001
        grid = torch.linspace(0, max(top, 1e-30), 4097, dtype=torch.float64)
        slope, at = torch.ones_like(grid), grid
        slopes = [1.0]
        for _ in range(steps - k):
            slope = slope * (a + 3 * b * at**2 + 5 * c * at**4)
            at = at * (a + b * at**2 + c * at**4)
            slopes.append(slope.abs().max().item())
        # (the step's own slope is in the sum above: what is left are the steps after it; X_0's conversion meets all of them)
        total += (e * x.norm().item() + 2.0**-27 * math.sqrt(x.numel())) * slopes[-2 if k else -1]
    return total


def schulz_halves(u: Tensor, steps: int = 5, coefficients=NEWTON_SCHULZ, eps: float = 1e-7, leave_out: str = "") -> Tensor:
    """One matrix's iteration as FP32 arithmetic on operands of two FP16 halves computes it, in some order of its sums: X, A and P
    times powers of two that keep a little more than their largest entries below FP16's largest number, each product hi hi + hi lo +
    lo hi with FP32 sums. How far this ends from the exact result is how far such an iteration may end. ``leave_out``: a
    product (``"gram"``, ``"square"`` or ``"apply"``) whose low halves are dropped, a mistake to be noticed."""
    a, b, c = coefficients
    grid = torch.linspace(0, 1, 257, dtype=torch.float64)
    most_x, most_p = 1.0, 0.0
    for k in range(steps):
        p = a + b * grid**2 + c * grid**4
        grid = grid * p
        most_p = max(most_p, p.abs().max().item())
        most_x = max(most_x, grid.abs().max().item()) if k + 1 < steps else most_x
    sx, sa, sp = (2.0 ** math.floor(math.log2(60000.0 / m)) for m in (1.1 * most_x, 1.25 * most_x**2, 1.05 * most_p))

    def halves(t, scale):
        t = t.float() * scale
        hi = t.half().float()
        return hi, (t - hi).half().float()

    def product(s, t, name):
        hi, lo = s[0] @ t[0], s[0] @ t[1] + s[1] @ t[0]
        return (hi if leave_out == name else hi + lo).double()

    tall = u.shape[0] > u.shape[1]
    u = (u.t() if tall else u).double()
    eye = torch.eye(u.shape[0], dtype=torch.float64, device=u.device)
    x = halves(u / (u.square().sum().sqrt() + eps), sx)
    for k in range(steps):
        gram = product(x, [t.t() for t in x], "gram") / sx**2
        half = halves(gram, sa)
        square = product(half, half, "square") / sa**2
        y = product(halves(a * eye + b * gram + c * square, sp), x, "apply") / (sp * sx)
        x = halves(y, sx)
    return y.t() if tall else y


def _sum_error(n: int) -> float:
    """Of FP32 sums of n terms, relative to the terms' magnitudes: independent roundings of 2^-24, four standard deviations."""
    return 4 * math.sqrt(n + 4) * 2.0**-24


def low_rank_adapters(base: Tensor | None, x: Tensor, a: Tensor, b: Tensor, index: Tensor, scale, d_out: Tensor | None = None,
                      half: float = 2.0**-16) -> dict[str, Tensor]:
    """``out`` and, with ``d_out``, the gradients ``x``, ``a``, ``b``, float64, row by row; ``*_error`` what FP32 sums and a
    product's operand kept to ``half`` may change. (``half`` covers operands of two 16-bit numbers, and 2^-20 of a row's largest
    for FP16 values that are small beside it.)"""
    k, n, (j, r) = x.shape[-1], b.shape[1], a.shape[:2]
    rows = x.double().reshape(-1, k)
    which = index.reshape(-1).repeat_interleave(rows.shape[0] // max(1, index.numel()))
    scales = (scale.double() if isinstance(scale, Tensor) else torch.full((j,), float(scale), dtype=torch.float64))
    d = None if d_out is None else d_out.double().reshape(-1, n)
    out = torch.zeros(rows.shape[0], n, dtype=torch.float64) if base is None else base.double().reshape(-1, n).clone()
    got = {"out": out, "out_error": 2.0**-24 * out.abs()}
    if d is not None:
        got |= {"x": torch.zeros_like(rows), "x_error": torch.zeros_like(rows)}
        got |= {name + kind: torch.zeros_like(t, dtype=torch.float64) for name, t in (("a", a), ("b", b)) for kind in ("", "_error")}

    def product(u, v, w, s, sums):  # s (u v^T) w^T, its error's bound, and the middle
        mid, terms = s * u @ v.t(), abs(s) * (u.abs() @ v.abs().t())
        off = (_sum_error(sums) + 2.0**-23) * terms + half * mid.abs() + 2.0**-20 * mid.abs().amax(1, keepdim=True)
        return mid @ w.t(), off @ w.abs().t() + _sum_error(r) * (mid.abs() @ w.abs().t()), mid, off

    for i in range(j):
        at = (which == i).nonzero().squeeze(1)
        if at.numel() == 0:
            continue
        xi, ai, bi, s = rows[at], a[i].double(), b[i].double(), scales[i].item()
        low, error, h, h_off = product(xi, ai, bi, s, k)
        got["out"][at] += low
        got["out_error"][at] += error + 2.0**-24 * low.abs()
        if d is None:
            continue
        di = d[at]
        got["x"][at], got["x_error"][at], t, t_off = product(di, bi.t(), ai.t(), s, n)
        m = at.numel()
        for name, u, u_off, v in (("a", t, t_off, xi), ("b", h, h_off, di)):
            total = u.t() @ v
            off = u_off.t() @ v.abs() + (_sum_error(m) + half) * (u.abs().t() @ v.abs())
            got[name][i], got[name + "_error"][i] = (total, off) if name == "a" else (total.t(), off.t())
    for name, shape in (("out", (*x.shape[:-1], n)), ("x", x.shape)):
        for kind in ("", "_error"):
            if name + kind in got:
                got[name + kind] = got[name + kind].reshape(shape)
    return got
