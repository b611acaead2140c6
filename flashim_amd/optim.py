"""An optimizer whose step for matrices is ``ops.muon_step_``: momentum, orthogonalized by Newton-Schulz products. Trains what
:mod:`flashim_amd.gated` and the low-rank adapters are made of, through :func:`flashim_amd.gated.train_step` or any other loop.
"""

from __future__ import annotations

from collections.abc import Iterable

import torch
from torch import Tensor
from torch.optim.adamw import adamw

from flashim_amd import ops
from flashim_amd.backends.hip.train import NEWTON_SCHULZ


class Muon(torch.optim.Optimizer):
    """Matrices, and parameters of three dimensions as stacks of matrices, each stepped by itself, take ``ops.muon_step_`` with
    an FP32 momentum; the others (norms' weights, biases) take AdamW with ``adam_lr``, ``adam_betas`` and ``adam_eps``. Parameters of
    more dimensions are refused: a convolution's weight is one matrix of its output channels by the rest, and not a stack of
    its kernels. Every option may differ by parameter group. All matrices of a group (on one GPU) are stepped in the same
    launches, and nothing waits for the GPU.

    A step in a captured graph needs one before it, which makes its state, and ``capturable=True`` where AdamW's parameters are
    among them: their step counts then lie on the GPU. Replays keep the options of the capture, its learning rates among them: a
    schedule that changes them needs a capture for each."""

    def __init__(self, params: Iterable, lr: float = 0.02, *, momentum: float = 0.95, nesterov: bool = True,
                 weight_decay: float = 0.0, adjust: str = "original", steps: int = 5, coefficients=NEWTON_SCHULZ,
                 eps: float = 1e-7, adam_lr: float = 1e-3, adam_betas: tuple[float, float] = (0.9, 0.95),
                 adam_eps: float = 1e-8, capturable: bool = False) -> None:
        if lr < 0 or adam_lr < 0 or weight_decay < 0 or not 0 <= momentum < 1:
            raise ValueError(f"Muon: lr {lr}, adam_lr {adam_lr}, weight_decay {weight_decay}, momentum {momentum}")
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, adjust=adjust,
                                      steps=steps, coefficients=coefficients, eps=eps, adam_lr=adam_lr, adam_betas=adam_betas,
                                      adam_eps=adam_eps, capturable=capturable))

    def add_param_group(self, param_group: dict) -> None:
        super().add_param_group(param_group)
        for p in self.param_groups[-1]["params"]:
            if p.ndim > 3:
                self.param_groups.pop()
                raise ValueError(f"Muon: a parameter of shape {tuple(p.shape)}: neither a matrix nor a stack of them (a convolution's "
                                 "weight would be one matrix, a view of two dimensions)")

    def load_state_dict(self, state_dict: dict) -> None:
        """As any optimizer's, but with states of its own (none is shared with the optimizer they came from), and momenta that
        stay FP32 beside parameters of 16 bits."""
        super().load_state_dict(state_dict)
        ids = [i for group in state_dict["param_groups"] for i in group["params"]]
        params = [p for group in self.param_groups for p in group["params"]]
        for i, p in zip(ids, params):
            saved = state_dict["state"].get(i, {})
            if p in self.state:
                self.state[p] = {k: v.clone() if isinstance(v, Tensor) else v for k, v in self.state[p].items()}
            if "momentum" in saved:
                self.state[p]["momentum"] = saved["momentum"].to(device=p.device, dtype=torch.float32, copy=True)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            with_grad = [p for p in group["params"] if p.grad is not None]
            matrices = [p for p in with_grad if p.ndim >= 2]
            if with_grad and with_grad[0].is_cuda and torch.cuda.is_current_stream_capturing():
                self._check_capture(group, with_grad)
            if matrices:
                ops.muon_step_(matrices, [p.grad for p in matrices], [self._momentum(p) for p in matrices], lr=group["lr"],
                               momentum=group["momentum"], nesterov=group["nesterov"], weight_decay=group["weight_decay"],
                               adjust=group["adjust"], steps=group["steps"], coefficients=group["coefficients"],
                               eps=group["eps"])
            self._adam(group, [p for p in with_grad if p.ndim < 2])
        return loss

    def _check_capture(self, group: dict, params: list[Tensor]) -> None:
        if not all(p in self.state for p in params):
            raise RuntimeError("Muon: a first step in a captured graph, whose replays would all start from its zeros")
        if not group["capturable"] and any(p.ndim < 2 for p in params):
            raise RuntimeError("Muon: AdamW's step counts would stand still in a captured graph; construct with capturable=True")

    def _momentum(self, p: Tensor) -> Tensor:
        state = self.state[p]
        if "momentum" not in state:
            state["momentum"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        return state["momentum"]

    def _adam(self, group: dict, params: list[Tensor]) -> None:
        if not params:
            return
        states = [self.state[p] for p in params]
        for p, state in zip(params, states):
            if not state:
                on = p.device if group["capturable"] else None
                state |= {"step": torch.zeros((), dtype=torch.float32, device=on), "exp_avg": torch.zeros_like(p),
                          "exp_avg_sq": torch.zeros_like(p)}
        beta1, beta2 = group["adam_betas"]
        adamw(params, [p.grad for p in params], [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states], [],
              [s["step"] for s in states], capturable=group["capturable"], amsgrad=False, beta1=beta1, beta2=beta2,
              lr=group["adam_lr"], weight_decay=group["weight_decay"], eps=group["adam_eps"], maximize=False)
