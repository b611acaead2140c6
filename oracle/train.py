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
