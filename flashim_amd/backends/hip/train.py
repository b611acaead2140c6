"""HIP impls of the training-step operators around the quantized layers. FlashIM is an inference library and has none of
them; here they train a channels-last block before it is quantized, and run it unquantized:

* ``group_norm_act``: group norm and activation of a channels-last map in one pass over it, with its gradients;
* ``gated_linear``: the gated feed-forward product, both projections, activation and product in one kernel, with its
  gradients;
* ``grad_norm`` and ``clip_grad_norm_``: the global norm of many gradients, and clipping by it.
"""

from __future__ import annotations

import math
from collections.abc import Sequence

import torch
from torch import Tensor

from flashim_amd import library
from flashim_amd.platforms import is_gfx950

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
_HALVES = (torch.bfloat16, torch.float16)
ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}  # the C ABI's codes
MAX_CHANNELS = 8192  # of group_norm_act


def group_norm_act(x: Tensor, num_groups: int, weight: Tensor | None = None, bias: Tensor | None = None, *,
                   eps: float = 1e-5, activation: str = "none") -> Tensor:
    """``act((x - mean) / sqrt(var + eps) * weight + bias)`` of a channels-last ``x`` ``[B, ..., C]``, mean and biased
    variance over the pixels and the ``C / num_groups`` channels of each (image, group). ``weight`` and ``bias`` ``[C]``
    in any float type; FP32 arithmetic, rounded once to ``x``'s type. A group with an infinity is NaN. Differentiable in
    ``x``, ``weight`` and ``bias``; second and forward-mode derivatives raise, here and in ``gated_linear``."""
    return library.group_norm_act(x, num_groups, weight, bias, eps, ACTIVATIONS[activation])[0]


def gated_linear(x: Tensor, w_gate: Tensor, w_up: Tensor, b_gate: Tensor | None = None, b_up: Tensor | None = None, *,
                 activation: str = "silu") -> Tensor:
    """``act(x Wg^T + bg) * (x Wu^T + bu)`` of ``x`` ``[..., K]`` and weights ``[H, K]`` in BF16 or FP16, biases ``[H]``
    in that type or FP32; FP32 sums, rounded once. Differentiable in every tensor: the backward pass computes the
    pre-activations again and rounds their gradients to ``x``'s type before the products that make the others."""
    return library.gated_linear(x, w_gate, w_up, b_gate, b_up, ACTIVATIONS[activation])


def grad_norm(grads: Sequence[Tensor], *, norm_type: float = 2.0) -> Tensor:
    """The norm (2 or ``math.inf``) over all elements of ``grads``: an FP32 value on their device, squares summed in 64
    bits. Nothing waits for the GPU."""
    return library.grad_norm(grads, float(norm_type))


def clip_grad_norm_(grads: Sequence[Tensor], max_norm: float, *, norm_type: float = 2.0,
                    out: Sequence[Tensor] | None = None, error_if_nonfinite: bool = False) -> Tensor:
    """Scales ``grads`` (no two of which overlap) by ``min(1, max_norm / (norm + 1e-6))`` in place, or into ``out`` (tensors
    of the same shapes that do not overlap the gradients, of any float type: BF16 gradients into the FP32 ones an optimizer
    reads), and returns the norm. A NaN norm makes every element NaN, as in ``torch.nn.utils.clip_grad_norm_``; with ``error_if_nonfinite``
    a norm that is not finite raises before anything is written (this waits for the GPU)."""
    with torch.no_grad():
        if error_if_nonfinite and not math.isfinite(library.grad_norm(grads, float(norm_type)).item()):
            raise RuntimeError(f"clip_grad_norm_: the gradients' norm of type {norm_type} is not finite")
        return library.clip_lists(grads, out, float(max_norm), float(norm_type))


# -- eligibility -------------------------------------------------------------------------------------------------------


def _vector(t: Tensor | None, n: int, like: Tensor, dtypes) -> bool:
    return t is None or (t.ndim == 1 and t.shape[0] == n and t.device == like.device and t.dtype in dtypes)


def eligible_group_norm_act(x, num_groups, weight=None, bias=None, *, eps=1e-5, activation="none") -> bool:
    return (
        isinstance(x, Tensor) and is_gfx950(x.device) and x.ndim >= 2 and x.dtype in _FLOATS
        and activation in ACTIVATIONS and 0 < x.shape[-1] <= MAX_CHANNELS
        and num_groups > 0 and x.shape[-1] % num_groups == 0
        and _vector(weight, x.shape[-1], x, _FLOATS) and _vector(bias, x.shape[-1], x, _FLOATS)
    )


def eligible_gated_linear(x, w_gate, w_up, b_gate=None, b_up=None, *, activation="silu") -> bool:
    return (
        isinstance(x, Tensor) and is_gfx950(x.device) and x.ndim >= 1 and x.dtype in _HALVES and x.shape[-1] > 0
        and activation in ACTIVATIONS
        and all(w.ndim == 2 and w.dtype == x.dtype and w.device == x.device and w.shape[1] == x.shape[-1]
                and w.shape[0] > 0 for w in (w_gate, w_up))
        and w_gate.shape == w_up.shape
        and all(_vector(b, w_gate.shape[0], x, (x.dtype, torch.float32)) for b in (b_gate, b_up))
        and (b_gate is None or b_up is None or b_gate.dtype == b_up.dtype)
    )


def _tensors(tensors) -> bool:
    return isinstance(tensors, (list, tuple)) and len(tensors) > 0 and all(issubclass(t, Tensor)
                                                                           for t in set(map(type, tensors)))


# The first gradient stands for the others here; the operators themselves look at each tensor's device, type and size, and
# raise NotImplementedError as a refused predicate does.


def eligible_grad_norm(grads, *, norm_type=2.0) -> bool:
    return _tensors(grads) and is_gfx950(grads[0].device) and grads[0].dtype in _FLOATS and norm_type in (2.0, math.inf)


def eligible_clip_grad_norm(grads, max_norm, *, norm_type=2.0, out=None, error_if_nonfinite=False) -> bool:
    return eligible_grad_norm(grads, norm_type=norm_type) and (out is None or (_tensors(out) and len(out) == len(grads)))
