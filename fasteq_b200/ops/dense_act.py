"""Dense layer with its epilogue, ``act(x @ weight.T + bias) + residual`` (``fasteq_product_forward``).

``dense`` followed by a bias, an activation and a residual is one product and three more passes over its result; here they are
part of the product's launch.  Where gradients will be asked for the forward also keeps ``act'``, so that the backward is one product for the
gradient of ``x`` and one for those of ``weight`` and ``bias``.  Launches besides: FP32 rows whose width is not a multiple of four are copied, FP32
weights of more than 256 channels to sum over are split beforehand, weight gradients of many rows add up partial sums, FP64 gradients multiply by
``act'`` first.  FP32 with the accuracy of FP32 products (three bf16 parts per operand on the tensor cores: 2-norm errors of 0.7 to 2.3e-7, 3.9e-7
where no signs cancel; sums that FP32 holds exactly are exact), FP64; any strides, up to 4,194,240 channels.  ``dense`` (3xTF32, errors near 1e-6) is
faster for wide layers without an epilogue.  Differentiable to every order: where a gradient is to be differentiated again the layer is taken
apart into bilinear products, which are one another's gradients.  Forward-mode differentiation is refused.

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
