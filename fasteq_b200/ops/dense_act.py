"""Dense layer with its epilogue, ``act(x @ weight.T + bias) + residual``, as one launch (``fasteq_product_forward``).

``dense`` followed by a bias, an activation and a residual is one product and three more passes over its result; here they are
part of the product.  Where gradients will be asked for the forward also keeps ``act'``, so that the backward is one launch for the
gradient of ``x`` and one (with its reduction) for those of ``weight`` and ``bias``.  FP32 with the accuracy of FP32 products (three
bf16 parts per operand on the tensor cores), FP64; any extents and strides.  Differentiable to every order: where a gradient is to be
differentiated again the layer is taken apart into bilinear products, which are one another's gradients.

Activations are those of the gate (``ops/gate.py``): ``None`` / ``"identity"``, ``"silu"``, ``"tanh"``, ``"sigmoid"``, ``"abs"``.
CUDA tensors only.
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import _front
from .gate import ACT_CODES


def act_code(name: str, activation) -> int:
    if activation not in ACT_CODES:
        raise ValueError(f"{name}: activation must be one of {[a for a in ACT_CODES if a]} or None, got {activation!r}")
    return ACT_CODES[activation]


def dense_act(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: Optional[str] = None,
              residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual``: ``x [..., K]``, ``weight [N, K]`` (a ``torch.nn.Linear`` weight), ``bias [N]``,
    ``residual [..., N]`` like the result."""
    return _front.lib().dense_act(x, weight, bias, act_code("dense_act", activation), residual)
