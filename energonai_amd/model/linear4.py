"""Projections with weights in 4 bits (``kernel.linear_w4``) in the place of ``torch.nn.Linear``.

The reference keeps its weights in 16 bits (energonai/model/mlp.py:15-25); a decode step of few rows is bound by reading them.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import nn

from ..kernel.w4 import W4Weight, linear_w4, w4_codes, w4_weight


class Linear4(nn.Module):
    """``act(x W^T + bias)`` with a weight in 4 bits.  The laid-out weight is kept in buffers, and saved and loaded with the module; a change of
    dtype changes its scales' type, to which the inputs' has to be equal."""

    def __init__(self, weight: W4Weight, bias: Optional[torch.Tensor] = None) -> None:
        super().__init__()
        self.in_features, self.out_features, self.group_size = weight.in_features, weight.out_features, weight.group_size
        self.register_buffer("codes", weight.codes)
        self.register_buffer("scales", weight.scales)
        self.register_buffer("zeros", weight.zeros)
        self.bias = None if bias is None else nn.Parameter(bias.detach().clone(), requires_grad=False)

    @classmethod
    def from_linear(cls, layer: nn.Linear, group_size: int = 128, zero_points: bool = False) -> "Linear4":
        """The layer with its weight rounded to 4 bits (``kernel.w4_codes``), on its GPU."""
        codes, scales, zeros = w4_codes(layer.weight.detach(), group_size, zero_points)
        return cls(w4_weight(codes, scales, zeros, group_size), layer.bias)

    def forward(self, x: torch.Tensor, activation: Optional[str] = None) -> torch.Tensor:
        w = W4Weight(self.codes, self.scales, self.zeros, self.out_features, self.in_features, self.group_size)
        return linear_w4(x, w, bias=self.bias, activation=activation)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, group_size={self.group_size}"


def quantize_linears(module: nn.Module, group_size: int = 128, zero_points: bool = False) -> nn.Module:
    """Replaces every ``torch.nn.Linear`` below ``module`` (fp16 or bf16, on a GPU) by a ``Linear4`` of it, in place; returns ``module``."""
    for name, child in list(module.named_children()):
        if type(child) is nn.Linear:
            setattr(module, name, Linear4.from_linear(child, group_size, zero_points))
        else:
            quantize_linears(child, group_size, zero_points)
    return module
