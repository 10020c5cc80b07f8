"""Experts: a node (or any row) is given to one or several of a set of matrices, as ``fast_fctp`` gives it to its species' one.

    plan = expert_plan(expert, num_experts)                       # who goes where: [tokens, slots] expert numbers, -1: to none
    rows = expert_gather(x, plan)                                 # [tokens, ...] -> [tokens * slots, ...] in the experts' order
    rows = expert_dense(rows, w1, plan, bias=b1, activation="silu")      # one product for all experts, w1 [experts, N, K]
    rows = expert_dense(rows, w2, plan, bias=b2)
    y = expert_combine(rows, plan, weight)                        # [tokens, ...] = sum over slots of weight * row

Everything stays on the device: the plan's offsets are read by the kernels, so the host waits for nothing and a step can be captured
in a CUDA graph.  Sums run over slots and rows in a fixed order (no atomics): the same inputs give the same bits.  Entries given to no
expert lie behind the experts' rows as zeros and take part in no sum and no gradient.  The weights are scalars of a row, so rows may hold
components of irreps; ``expert_dense`` mixes channels, its rows' components ``[rows, components, K]`` share their expert's matrix.
Float32 and float64, differentiable to every order (forward-mode differentiation is refused).  CUDA tensors only.
"""
from __future__ import annotations

import ctypes as C
import functools
from typing import Optional

import torch

from .. import _cabi, _front
from .dense_act import act_code

__all__ = ["ExpertPlan", "expert_plan", "expert_gather", "expert_dense", "expert_combine", "expert_device_status"]


class ExpertPlan:
    """Order of the entries ``(token, slot)`` by expert.  ``position [tokens, slots]``: the entry's row; ``offsets [num_experts + 1]``: expert
    ``e`` has rows ``offsets[e]`` to ``offsets[e + 1]``, those from ``offsets[-1]`` on have none (both int32, on the device; to be read: calls and
    gradients refuse a plan whose tensors were changed in place)."""

    def __init__(self, native):
        self._native = native
        self.tokens, self.slots, self.num_experts = native.shape
        self.rows = self.tokens * self.slots

    @functools.cached_property
    def position(self) -> torch.Tensor:
        return self._native.position

    @functools.cached_property
    def offsets(self) -> torch.Tensor:
        return self._native.offsets


def expert_device_status() -> int:
    """Reads and clears the status word of the plans (synchronises): 0, or 2 = an expert number was not below ``num_experts``, or a
    position not among the rows."""
    lib, v = _cabi.core(), C.c_int32(0)
    _cabi.check(lib.fasteq_expert_device_status(C.byref(v)), lib, "fasteq_expert_device_status")
    return int(v.value)


def expert_plan(expert: torch.Tensor, num_experts: int) -> ExpertPlan:
    """``expert [tokens, slots]`` (or ``[tokens]``: one slot), int32 or int64.  Negative numbers mean no expert; numbers from ``num_experts``
    on are treated like them and reported by ``fasteq_b200.status.device_status``."""
    return ExpertPlan(_front.lib().expert_plan(expert, num_experts))


def _order(name: str, plan: ExpertPlan):
    if not isinstance(plan, ExpertPlan):
        raise TypeError(f"{name}: plan must be an ExpertPlan, got {type(plan).__name__}")
    return plan._native


def expert_gather(x: torch.Tensor, plan: ExpertPlan) -> torch.Tensor:
    """``x [tokens, ...]`` to ``[tokens * slots, ...]`` in the experts' order (zeros for entries of no expert)."""
    return _front.lib().expert_gather(x, _order("expert_gather", plan))


def expert_combine(rows: torch.Tensor, plan: ExpertPlan, weight: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``y[t] = sum_s weight[t, s] * rows[position[t, s]]``: ``rows [tokens * slots, ...]`` in the experts' order, ``weight [tokens, slots]``
    (``[tokens]`` with one slot; ``None``: ones)."""
    return _front.lib().expert_combine(rows, weight, _order("expert_combine", plan))


def expert_dense(rows: torch.Tensor, weight: torch.Tensor, plan: ExpertPlan, bias: Optional[torch.Tensor] = None,
                 activation: Optional[str] = None) -> torch.Tensor:
    """``act(rows[r] @ weight[e(r)].T + bias[e(r)])`` for rows in the experts' order, ``[tokens * slots, ..., K]``; ``weight [num_experts, N, K]``,
    ``bias [num_experts, N]``, activations as in ``dense_act``.  Rows of no expert come out as zeros."""
    return _front.lib().expert_dense(rows, weight, _order("expert_dense", plan), bias, act_code("expert_dense", activation))
