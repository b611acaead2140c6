"""A channels-last gated block, trained on the differentiable operators and then run quantized on the package's static
convolutions: the use that ``ops.group_norm_act``, ``ops.gated_linear`` and ``ops.clip_grad_norm_`` are made for.

``y = x + act(n Wg^T + bg) * (n Wu^T + bu) Wd^T + bd``, ``n`` the group norm of ``x`` ``[B, H, W, C]`` (BF16 or FP16).

Training: :class:`GatedBlock` is an ordinary module; :func:`train_step` takes its gradients, clips them by their global norm
and steps the optimizer. Inference: :class:`QuantizedGatedBlock` keeps the norm and the gated product, quantizes the hidden
map with static scales from one calibration pass, and contracts it with the INT8 or MXFP8 1x1 convolution and its fused
residual, as the refiner blocks (:mod:`flashim_amd.blocks`) do.

Adapting: :class:`Adapters` are low-rank changes of the contraction, one of them for each image of a batch (``index``).
:class:`AdaptedGatedBlock` trains them beside a frozen block (``train_step`` with :class:`flashim_amd.optim.Muon`, say), and
:class:`QuantizedGatedBlock` takes them beside its INT8 or MXFP8 contraction: many requests' adapters at once, one set of
quantized weights.
"""

from __future__ import annotations

from collections.abc import Callable

import torch
import torch.nn.functional as F
from torch import Tensor, nn

from flashim_amd import ops, quant

_POINTWISE = (1, 1, 1, 1, 0, 0, 1, 1)


class GatedBlock(nn.Module):
    """``channels`` wide, ``hidden`` inside, ``groups`` in the norm; parameters in ``dtype``, those of the norm in FP32."""

    def __init__(self, channels: int, hidden: int, groups: int, *, activation: str = "silu",
                 dtype: torch.dtype = torch.bfloat16, device="cuda", generator: torch.Generator | None = None) -> None:
        super().__init__()
        self.groups, self.activation = groups, activation

        def matrix(rows: int, cols: int) -> nn.Parameter:
            return nn.Parameter((torch.randn(rows, cols, generator=generator) * cols ** -0.5).to(device=device, dtype=dtype))

        def vector(n: int, value: float = 0.0, kind: torch.dtype = dtype) -> nn.Parameter:
            return nn.Parameter(torch.full((n,), value, dtype=kind, device=device))

        self.norm_weight, self.norm_bias = vector(channels, 1.0, torch.float32), vector(channels, 0.0, torch.float32)
        self.w_gate, self.w_up = matrix(hidden, channels), matrix(hidden, channels)
        self.b_gate, self.b_up = vector(hidden), vector(hidden)
        self.w_down, self.b_down = matrix(channels, hidden), vector(channels)

    def hidden(self, x: Tensor) -> Tensor:
        normed = ops.group_norm_act(x, self.groups, self.norm_weight, self.norm_bias)
        return ops.gated_linear(normed, self.w_gate, self.w_up, self.b_gate, self.b_up, activation=self.activation)

    def forward(self, x: Tensor) -> Tensor:
        return x + F.linear(self.hidden(x), self.w_down, self.b_down)


def train_step(module: nn.Module, optimizer: torch.optim.Optimizer, loss: Callable[[], Tensor],
               max_norm: float) -> tuple[Tensor, Tensor]:
    """One step: ``loss()`` and its gradients, clipped in place to a global norm of ``max_norm``. Returns the loss and the
    norm before clipping (0 where no parameter of ``module`` has a gradient), both on the GPU (nothing waits for it)."""
    optimizer.zero_grad(set_to_none=True)
    value = loss()
    value.backward()
    grads = [p.grad for p in module.parameters() if p.grad is not None]
    norm = ops.clip_grad_norm_(grads, max_norm) if grads else torch.zeros((), device=value.device)
    optimizer.step()
    return value.detach(), norm


class Adapters(nn.Module):
    """``count`` adapters of a block's contraction, ``scale (h A_j^T) B_j^T`` beside ``h Wd^T``: ``a`` random, ``b`` zero (no
    change) at first."""

    def __init__(self, block: GatedBlock, count: int, rank: int, *, scale: float = 1.0,
                 generator: torch.Generator | None = None) -> None:
        super().__init__()
        channels, hidden = block.w_down.shape
        like = dict(dtype=block.w_down.dtype, device=block.w_down.device)
        self.a = nn.Parameter((torch.randn(count, rank, hidden, generator=generator) * hidden ** -0.5).to(**like))
        self.b = nn.Parameter(torch.zeros(count, channels, rank, **like))
        self.scale = scale

    def forward(self, base: Tensor, hidden: Tensor, index: Tensor) -> Tensor:
        """``base`` and each image's adapter of ``hidden``; ``index`` ``[B]``, outside ``[0, count)`` for none."""
        return ops.low_rank_adapters(base, hidden, self.a, self.b, index, scale=self.scale)


class AdaptedGatedBlock(nn.Module):
    """``block``, whose parameters this freezes, with ``adapters`` that train."""

    def __init__(self, block: GatedBlock, adapters: Adapters) -> None:
        super().__init__()
        self.block, self.adapters = block.requires_grad_(False), adapters

    def forward(self, x: Tensor, index: Tensor) -> Tensor:
        hidden = self.block.hidden(x)
        return self.adapters(x + F.linear(hidden, self.block.w_down, self.block.b_down), hidden, index)


class QuantizedGatedBlock:
    """A trained block with its contraction in ``preset`` ``"int8"`` or ``"mxfp8"``; ``sample`` gives the hidden map's static
    scale. BF16, ``hidden`` a multiple of 32. A call with ``adapters`` and ``index`` ``[B]`` adds each image's adapter, from the
    hidden map as it was before its quantization."""

    def __init__(self, block: GatedBlock, preset: str, sample: Tensor) -> None:
        if preset not in ("int8", "mxfp8"):
            raise ValueError(f"unknown preset {preset!r}")
        self.block, self.preset = block, preset
        with torch.no_grad():
            hidden = block.hidden(sample)
            if preset == "mxfp8":
                self.weight = quant.QuantizedWeight.from_float(block.w_down.detach())
                self.scale = quant.calibrate_block32_exponent(hidden)
            else:
                self.weight = quant.weight_scales_and_values(block.w_down.detach())
                self.scale = (hidden.float().abs().amax() / quant.INT8_MAX).clamp_min(1e-8).reshape(())

    @torch.no_grad()
    def __call__(self, x: Tensor, adapters: Adapters | None = None, index: Tensor | None = None) -> Tensor:
        if (adapters is None) != (index is None):
            raise ValueError("adapters come with an index of them")
        hidden, bias = self.block.hidden(x), self.block.b_down.detach()
        if self.preset == "mxfp8":
            q = ops.quantize_mxfp8(hidden, self.scale)
            out = ops.mxfp8_conv2d(q.values, self.scale, self.weight.values, self.weight.scale_exponent, bias, *_POINTWISE,
                                   residual=x)
        else:
            codes, weight_scale = self.weight
            q = ops.quantize_int8(hidden, self.scale)
            out = ops.int8_conv2d(q.values, codes, self.scale, weight_scale, bias, *_POINTWISE, residual=x)
        return out if adapters is None else adapters(out, hidden, index)
