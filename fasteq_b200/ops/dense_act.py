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


def check_operands(name: str, **operands) -> None:
    """CUDA tensors of one device and one type, float32 or float64 (``None``: left out)."""
    first = None
    for what, t in operands.items():
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name}: {what} must be a tensor, got {type(t).__name__}")
        if not t.is_cuda:
            raise RuntimeError(f"{name}: {what} must be a CUDA tensor: fasteq_b200 has no CPU path")
        if t.dtype not in (torch.float32, torch.float64):
            raise ValueError(f"{name}: only float32 and float64 are supported; {what} is {t.dtype}")
        first = first if first is not None else t
        if t.dtype != first.dtype or t.device != first.device:
            raise ValueError(f"{name}: all operands must have one dtype and one device; {what} is {t.dtype} on {t.device}, not {first.dtype} on {first.device}")


def dense_act(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: Optional[str] = None,
              residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual``: ``x [..., K]``, ``weight [N, K]`` (a ``torch.nn.Linear`` weight), ``bias [N]``,
    ``residual [..., N]`` like the result."""
    code = act_code("dense_act", activation)
    check_operands("dense_act", x=x, weight=weight, bias=bias, residual=residual)
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"dense_act: x [..., K] and weight [N, K] expected, got {tuple(x.shape)} and {tuple(weight.shape)}")
    if bias is not None and bias.shape != weight.shape[:1]:
        raise ValueError(f"dense_act: bias must be [{weight.shape[0]}], got {tuple(bias.shape)}")
    if residual is not None and residual.shape != (*x.shape[:-1], weight.shape[0]):
        raise ValueError(f"dense_act: residual must have the result's shape {(*x.shape[:-1], weight.shape[0])}, got {tuple(residual.shape)}")
    return _front.lib().product_layer(x, weight, bias, residual, None, 1, code)
