"""Projections with weights in 4 bits (``kernel.linear_w4``) in the place of ``torch.nn.Linear``.

The reference keeps its weights in 16 bits (energonai/model/mlp.py:15-25); a decode step of few rows is bound by reading them.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import nn

from .. import _lib
from ..kernel.w4 import W4Weight, check_w4_codes, linear_w4, w4_codes, w4_weight


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
    """Replaces every ``torch.nn.Linear`` below ``module`` (fp16 or bf16, on a GPU) by a ``Linear4`` of it, in place; returns ``module``.  One that
    several modules share, or that has several names, becomes one that they share.  Where one cannot be replaced, none is."""
    places = {}                 # the layer -> (module, name) of all its places
    for parent in module.modules():
        for name, child in parent._modules.items():
            if type(child) is nn.Linear:
                places.setdefault(child, []).append((parent, name))
    for layer in places:
        check_w4_codes("quantize_linears", layer.weight.detach(), group_size)
        _lib.require_gpu(layer.weight, "weight", contiguous=False)
    child = None
    while places:               # the last one that holds a layer's 16-bit weight lets it go before the next is turned
        layer, at = places.popitem()
        small = Linear4.from_linear(layer, group_size, zero_points)
        for parent, name in at:
            setattr(parent, name, small)
    return module
