"""Weights in 4 bits with a scale for each group of neighbouring input channels, and the products with them.

``W[n, k] = (code[n, k] - zero[n, g]) * scale[n, g]`` with codes 0 .. 15, ``g = k // group_size`` and zero points 0 .. 255 (without them 8).  A
decode step of few rows is bound by the bytes of its weights, and these are a quarter of what 16 bits are.  The reference has weights in 16 bits
alone (energonai/kernel/cuda_native/linear_func.py:11-32).
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from .. import _lib

_TYPES = (torch.float16, torch.bfloat16)
_GROUPS = (32, 64, 128)
_FARTHEST = 1 << 21          # elements from row to row that en_linear_w4 takes
_ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "gelu_tanh": 2, "gelu": 3}


class W4Weight(NamedTuple):
    """A weight as ``linear_w4`` reads it (made by ``w4_weight`` or ``w4_quantize``)."""
    codes: torch.Tensor                 # uint8 [tiles of 16 rows, tiles of 128 channels, 1024]
    scales: torch.Tensor                # fp16 or bf16 [tiles of 16 rows, tiles of 128 channels, 16, groups of a tile]
    zeros: Optional[torch.Tensor]       # uint8, as many; None: 8
    out_features: int
    in_features: int
    group_size: int


def _struct(who: str, w) -> _lib.W4:
    if not isinstance(w, W4Weight):
        raise RuntimeError(f"{who}: weight must be a W4Weight")
    N, K, G = int(w.out_features), int(w.in_features), int(w.group_size)
    groups = int(_lib.fn.en_w4_groups(N, K, G))
    for t, n in ((w.codes, "codes"), (w.scales, "scales"), (w.zeros, "zeros")):
        if t is None and n == "zeros":
            continue
        _lib.require_gpu(t, n)
        if t.device != w.codes.device or t.numel() != (int(_lib.fn.en_w4_codes_bytes(N, K)) if n == "codes" else groups) \
                or t.dtype not in (_TYPES if n == "scales" else (torch.uint8,)):
            raise RuntimeError(f"{who}: the weight's {n} are not those of {N} x {K} in groups of {G}")
    return _lib.W4(w.codes.data_ptr(), w.scales.data_ptr(), _lib.ptr(w.zeros) or None, N, K, G, _lib.dtype_tag(w.scales, who))


def w4_weight(codes, scales, zeros=None, group_size: int = 128) -> W4Weight:
    """Lays out a weight given as ``codes`` uint8 ``[dout, din / 2]`` (channel 2i in the lower four bits of byte i), ``scales`` fp16 or bf16 ``[dout,
    ceil(din / group_size)]`` and ``zeros`` uint8 of that shape, or ``None`` for 8.  ``din`` a multiple of 8, groups of 32, 64 or 128."""
    who = "w4_weight"
    for t, n in ((codes, "codes"), (scales, "scales"), (zeros, "zeros")):
        if t is not None or n != "zeros":
            _lib.require_gpu(t, n)
            if t.device != codes.device:
                raise RuntimeError(f"{who}: {n} must be on the codes' device")
    if codes.dim() != 2 or codes.dtype != torch.uint8 or codes.shape[0] < 1 or codes.shape[1] < 4 or codes.shape[1] % 4:
        raise RuntimeError(f"{who}: codes must be uint8 [dout, din / 2] with din a multiple of 8")
    if group_size not in _GROUPS:
        raise RuntimeError(f"{who}: group_size must be one of {_GROUPS}")
    N, K = codes.shape[0], 2 * codes.shape[1]
    shape = (N, -(-K // group_size))
    if scales.shape != shape or scales.dtype not in _TYPES or (zeros is not None and (zeros.shape != shape or zeros.dtype != torch.uint8)):
        raise RuntimeError(f"{who}: scales must be float16 or bfloat16 and zeros uint8, {list(shape)} each")
    tiles, steps = -(-N // 16), -(-K // 128)
    per = (tiles, steps, 16, 128 // group_size)
    w = W4Weight(torch.empty((tiles, steps, 1024), dtype=torch.uint8, device=codes.device), torch.empty(per, dtype=scales.dtype, device=codes.device),
                 None if zeros is None else torch.empty(per, dtype=torch.uint8, device=codes.device), N, K, int(group_size))
    with _lib.device_guard(codes):
        _lib.check(_lib.fn.en_w4_pack(codes.data_ptr(), scales.data_ptr(), _lib.ptr(zeros) or None, ctypes.byref(_struct(who, w)), _lib.stream_of(codes)), who)
    return w


def check_w4_codes(who: str, weight, group_size: int) -> None:
    """Raises where ``w4_codes`` has no codes for a weight."""
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or weight.dtype not in _TYPES or weight.shape[1] % 8 or weight.numel() == 0:
        raise RuntimeError(f"{who}: weight must be a float16 or bfloat16 [dout, din] tensor with din a multiple of 8")
    if group_size not in _GROUPS:
        raise RuntimeError(f"{who}: group_size must be one of {_GROUPS}")


@torch.no_grad()
def w4_codes(weight, group_size: int = 128, zero_points: bool = False):
    """``(codes, scales, zeros)`` of a ``[dout, din]`` weight, as ``w4_weight`` takes them, rounded to the nearest.  Without zero points a
    group's largest magnitude is code 0 (-8) or, where it is positive, 15 (7) or nearer to 0, whichever scale leaves the smaller squares; with them
    the group's range, and 0, are its codes 0 and 15.  A group without values has scale 0."""
    who = "w4_codes"
    check_w4_codes(who, weight, group_size)
    N, K = weight.shape
    groups = -(-K // group_size)
    w = torch.nn.functional.pad(weight.float(), (0, groups * group_size - K)).view(N, groups, group_size)

    def coded(scale, zero):
        by = torch.where(scale > 0, 1 / scale.clamp(min=1e-38), 0.0)[..., None]
        return ((w * by).round() + zero[..., None]).clamp(0, 15)

    if zero_points:
        low, high = w.amin(-1).clamp(max=0), w.amax(-1).clamp(min=0)
        scale = ((high - low) / 15).to(weight.dtype)
        zeros = torch.where(scale > 0, (-low / scale.float().clamp(min=1e-38)).round(), 0.0).clamp(0, 15)
        codes = coded(scale.float(), zeros)
    else:
        top = w.abs().amax(-1)
        eight = torch.full_like(top, 8.0)
        best = None
        for steps in (8.0, 7.5, 7.0):
            scale = (top / steps).to(weight.dtype)
            c = coded(scale.float(), eight)
            off = (((c - 8) * scale.float()[..., None] - w) ** 2).sum(-1)
            if best is None:
                best = [off, c, scale]
            else:
                less = off < best[0]
                best = [torch.where(less, off, best[0]), torch.where(less[..., None], c, best[1]), torch.where(less, scale, best[2])]
        codes, scale, zeros = best[1], best[2], None
    c = codes.view(N, -1)[:, :K].to(torch.uint8)
    return (c[:, 0::2] | c[:, 1::2] << 4).contiguous(), scale.contiguous(), None if zeros is None else zeros.to(torch.uint8).contiguous()


def w4_quantize(weight, group_size: int = 128, zero_points: bool = False) -> W4Weight:
    """``w4_weight`` of the ``w4_codes`` of a ``[dout, din]`` weight on the GPU."""
    _lib.require_gpu(weight, "weight", contiguous=False)
    return w4_weight(*w4_codes(weight, group_size, zero_points), group_size=group_size)


def linear_w4(inputs, weight, bias=None, activation: Optional[str] = None):
    """``linear`` with a weight in 4 bits: ``act(inputs[..., din] @ W[dout, din]^T + bias)`` -> ``[..., dout]``, fp16 or bf16 as the weight's
    scales are.  Sums are fp32; up to 64 rows no weight is rounded, from there on each is, to the inputs' type: a row's result differs, within those roundings, with
    how many rows it comes among, and so may what is chosen from near ties.  Up to 64 rows a row that holds an infinity may give NaN where the formula has an infinity
    (zero points are taken off the sums).  ``activation``: ``"relu"``, ``"gelu_tanh"`` or ``"gelu"``.  Up to 2^20 rows and 2^21 features.  Like the other operators of this package it is for inference: no gradient flows through it."""
    who = "linear_w4"
    if type(weight) is W4Weight and activation in _ACTIVATIONS:
        y = _lib.front.linear_w4(inputs, weight, bias, _ACTIVATIONS[activation])
        if y is not None:
            return y
    w = _struct(who, weight)
    _lib.require_gpu(inputs, "inputs", contiguous=False)
    if inputs.dim() < 1 or inputs.shape[-1] != w.in_features or inputs.dtype != weight.scales.dtype or inputs.device != weight.codes.device:
        raise RuntimeError(f"{who}: inputs must be [..., {w.in_features}] of the scales' dtype on the weight's device")
    if activation not in _ACTIVATIONS:
        raise RuntimeError(f"{who}: activation must be one of {sorted(k for k in _ACTIVATIONS if k)}")
    if bias is not None:
        _lib.require_gpu(bias, "bias")
        if bias.shape != (w.out_features,) or bias.dtype != inputs.dtype or bias.device != inputs.device:
            raise RuntimeError(f"{who}: bias must be [{w.out_features}] of the inputs' dtype on their device")
    x = inputs if inputs.dim() == 2 else inputs.reshape(-1, w.in_features)
    if x.shape[0] > 1 and (x.stride(0) % 8 or not w.in_features <= x.stride(0) <= _FARTHEST) or x.stride(1) != 1:
        x = x.contiguous()
    if x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
    rows = x.shape[0]
    out = torch.empty((*inputs.shape[:-1], w.out_features), dtype=inputs.dtype, device=inputs.device)
    need = int(_lib.fn.en_linear_w4_workspace_bytes(rows, w.out_features, w.in_features))
    workspace = torch.empty(need, dtype=torch.uint8, device=inputs.device)
    with _lib.device_guard(inputs):
        _lib.check(_lib.fn.en_linear_w4(x.data_ptr(), rows, x.stride(0) if rows > 1 else w.in_features, ctypes.byref(w), _lib.ptr(bias) or None,
                                        _ACTIVATIONS[activation], out.data_ptr(), _lib.ptr(workspace) or None, need, _lib.stream_of(inputs)), who)
    return out
