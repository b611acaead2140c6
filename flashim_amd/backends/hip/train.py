"""HIP impls of the training-step operators around the quantized layers. FlashIM is an inference library and has none of
them; here they train a channels-last block before it is quantized, and run it unquantized:

* ``group_norm_act``: group norm and activation of a channels-last map in one pass over it, with its gradients;
* ``gated_linear``: the gated feed-forward product, both projections, activation and product in one kernel, with its
  gradients;
* ``grad_norm`` and ``clip_grad_norm_``: the global norm of many gradients, and clipping by it;
* ``orthogonalize`` and ``muon_step_``: matrices orthogonalized by Newton-Schulz products, and the optimizer step made of them;
* ``low_rank_adapters``: low-rank adapters of many requests beside a shared projection, with their gradients.
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
_INDEX = (torch.int32, torch.int64)
ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}  # the C ABI's codes
MAX_CHANNELS = 8192  # of group_norm_act
MAX_RANK = 128  # of low_rank_adapters
NEWTON_SCHULZ = (3.4445, -4.7750, 2.0315)  # orthogonalize's coefficients: steepest at 0, within 0.7 .. 1.2 near 1
ADJUST = {"original": 0, "match_rms": 1, "none": 2}  # muon_step_'s factors


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


def orthogonalize(g: Tensor, *, steps: int = 5, coefficients: Sequence[float] = NEWTON_SCHULZ, eps: float = 1e-7,
                  out_dtype: torch.dtype | None = None) -> Tensor:
    """Each matrix of ``g`` ``[..., rows, cols]`` with its singular values brought near 1: ``X = g / (|g| + eps)`` (the Frobenius
    norm), then ``steps`` times ``A = X X^T``, ``X = (a I + b A + c A^2) X`` with ``coefficients = (a, b, c)`` (from the right
    for tall matrices). Products to FP32's precision, rounded once to ``out_dtype`` (``g``'s); values of X below
    2^-27 may count as zero (all of them where the norm is that far below ``eps``). Raises ``UnsupportedShape`` for
    coefficients by which a singular value of at most 1 passes 6 on its way. Not differentiable."""
    a, b, c = coefficients
    return library.orthogonalize(g, steps, a, b, c, eps, out_dtype)


def muon_step_(params: Sequence[Tensor], grads: Sequence[Tensor], momenta: Sequence[Tensor], *, lr: float, momentum: float = 0.95,
               nesterov: bool = True, weight_decay: float = 0.0, adjust: str = "original", steps: int = 5,
               coefficients: Sequence[float] = NEWTON_SCHULZ, eps: float = 1e-7) -> None:
    """One step of ``params`` (matrices, or stacks of them in the leading dimensions, each matrix by itself), in place:
    ``m = momentum m + g``, ``u = g + momentum m`` (``nesterov``) or ``m``,
    ``p = p (1 - lr weight_decay) - lr f orthogonalize(u)``. ``momenta`` FP32, the others of any float type. ``f`` by
    ``adjust``: ``"original"`` sqrt(max(1, rows / cols)), ``"match_rms"`` 0.2 sqrt(max(rows, cols)), ``"none"`` 1. No
    parameter or momentum shares an element with another tensor of the call (else ``ValueError``). Nothing waits for the GPU; a
    captured graph keeps ``lr`` and the other numbers."""
    a, b, c = coefficients
    with torch.no_grad():
        library.muon_step_(params, grads, momenta, lr, momentum, nesterov, weight_decay, ADJUST[adjust], steps, a, b, c, eps)


def low_rank_adapters(base: Tensor | None, x: Tensor, a: Tensor, b: Tensor, index: Tensor, *,
                      scale: float | Tensor = 1.0) -> Tensor:
    """``base + s_j (x A_j^T) B_j^T`` for each row of ``x`` ``[..., K]``, beside a shared projection's output ``base``
    ``[..., N]`` (None: zeros) of any kind. ``a`` ``[J, R, K]`` and ``b`` ``[J, N, R]`` (rank ``R`` at most 128), all BF16 or
    all FP16; ``index`` (int32 or int64) has the shape of some of ``x``'s leading dimensions and names each entry's adapter:
    one a row, or one an image, or one for all. A value outside ``[0, J)`` means none: the row keeps ``base``. ``scale``: a
    number, or FP32 ``[J]``. FP32 sums, rounded once. Differentiable in ``base``, ``x``, ``a`` and ``b``. Past 512 rows
    an index by row is several times as fast sorted as in random order."""
    scales, factor = (scale, 1.0) if isinstance(scale, Tensor) else (None, float(scale))
    save = torch.is_grad_enabled() and (a.requires_grad or b.requires_grad)
    return library.low_rank_adapters(base, x, a, b, index, scales, factor, save)[0]


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


def _polynomial(steps, coefficients, eps) -> bool:
    return 1 <= steps <= 100 and len(coefficients) == 3 and eps >= 0


def eligible_orthogonalize(g, *, steps=5, coefficients=NEWTON_SCHULZ, eps=1e-7, out_dtype=None) -> bool:
    return (isinstance(g, Tensor) and is_gfx950(g.device) and g.ndim >= 2 and g.dtype in _FLOATS
            and (out_dtype is None or out_dtype in _FLOATS) and _polynomial(steps, coefficients, eps))


def eligible_muon_step(params, grads, momenta, *, lr, momentum=0.95, nesterov=True, weight_decay=0.0, adjust="original", steps=5,
                       coefficients=NEWTON_SCHULZ, eps=1e-7) -> bool:
    return (all(_tensors(t) and len(t) == len(params) for t in (params, grads, momenta)) and is_gfx950(params[0].device)
            and params[0].dtype in _FLOATS and adjust in ADJUST and _polynomial(steps, coefficients, eps))


def eligible_low_rank_adapters(base, x, a, b, index, *, scale=1.0) -> bool:
    # (each attribute read once: a call's launch is no longer than this)
    if not (isinstance(x, Tensor) and isinstance(a, Tensor) and isinstance(b, Tensor) and isinstance(index, Tensor)):
        return False
    device, dtype = x.device, x.dtype
    if not is_gfx950(device) or dtype not in _HALVES or a.dtype is not dtype or b.dtype is not dtype:
        return False
    xs, sa, sb, si = x.shape, a.shape, b.shape, index.shape
    if len(sa) != 3 or len(sb) != 3 or not 1 <= len(xs) > len(si) or si != xs[:len(si)]:
        return False
    (adapters, rank, k), n = sa, sb[1]
    if xs[-1] != k or sb[0] != adapters or sb[2] != rank or not (0 < rank <= MAX_RANK and k > 0 and n > 0 and adapters > 0):
        return False
    if a.device != device or b.device != device or index.device != device or index.dtype not in _INDEX:
        return False
    if base is not None and not (isinstance(base, Tensor) and base.dtype is dtype and base.device == device
                                 and base.shape == xs[:-1] + (n,)):
        return False
    return not isinstance(scale, Tensor) or _vector(scale, adapters, x, (torch.float32,))
