"""Rotary positions and norms of heads, on packed rows and on a decode step's way into a paged cache.

The reference's models learn their positions (examples/gpt/gpt.py, examples/opt); models that rotate their queries and keys instead
need these between the projection and the attention.  A head's row goes through in fp32 and is rounded once:

    y = x * rsqrt(mean(x^2) + eps) * weight          where there is a weight
    (a, b) -> (a cos - b sin, b cos + a sin)         for the pairs of its first ``rotary_dim`` channels, at the row's position

with a, b = channels i and i + rotary_dim / 2, or 2i and 2i + 1 (``interleaved``).
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from .. import _lib
from ..seqinfo import SeqInfo, seq_info
from .attention import _overflow, _page_table, _pool


def rotary_table(max_positions: int, rotary_dim: int, base: float = 10000.0, device=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(cos, sin)``, float32 ``[max_positions, rotary_dim / 2]`` each, of the angles ``position * base ** (-2 i / rotary_dim)``, which are
    computed in 64 bits.  A model with other frequencies passes its own two tables."""
    if max_positions < 1 or rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_table: max_positions must be positive and rotary_dim a positive even number")
    inv = float(base) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    angles = torch.arange(max_positions, dtype=torch.float64)[:, None] * inv
    device = torch.device("cuda") if device is None else device
    return angles.cos().float().to(device), angles.sin().float().to(device)


def _rows(t, name: str, who: str) -> torch.Tensor:
    _lib.require_gpu(t, name, contiguous=False)
    if t.dim() != 3 or (t.shape[2] > 1 and t.stride(2) != 1):
        raise RuntimeError(f"{who}: {name} must be a [rows, head, size_per_head] view with contiguous channels")
    return t


def _span(t: torch.Tensor):
    return t.data_ptr(), t.data_ptr() + (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) * t.element_size() if t.numel() else t.data_ptr()


def _apart(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two sets of rows share no memory: one lies behind the other as a whole, in each token, or in each head's place."""
    (a0, a1), (b0, b1) = _span(a), _span(b)
    if a0 >= b1 or b0 >= a1:
        return True
    if b0 < a0:
        a, b, a0, b0 = b, a, b0, a0
    off, D, (token, head) = (b0 - a0) // a.element_size(), a.shape[2], a.stride()[:2]
    if b.stride(0) == token and token > 0:
        wide = [(t.shape[1] - 1) * t.stride(1) + D for t in (a, b)]
        if wide[0] <= off % token and off % token + wide[1] <= token:
            return True
    single = a.shape[0] == 1 and b.shape[0] == 1
    return head > 0 and b.stride(1) == head and (single or (b.stride(0) == token and token % head == 0)) and D <= off % head <= head - D


def _not_over(who: str, inputs, outs) -> None:
    """Refuses results that would be written over rows still to be read: each may be its own input, or lie apart from all of them."""
    for o in outs:
        inner, outer = sorted((s, n) for n, s in zip(o.shape[:2], o.stride()[:2]))
        if o.numel() and ((inner[1] > 1 and inner[0] < o.shape[2]) or (outer[1] > 1 and outer[0] < (inner[1] - 1) * inner[0] + o.shape[2])):
            raise RuntimeError(f"{who}: the rows of out must not overlap")
    for i, o in enumerate(outs):
        for j, t in enumerate(inputs):
            own = i == j and o.data_ptr() == t.data_ptr() and o.stride() == t.stride()
            if not own and not _apart(o, t):
                raise RuntimeError(f"{who}: out must be q and k themselves, which share no memory then, or lie apart from them")
    if len(outs) == 2 and not _apart(*outs):
        raise RuntimeError(f"{who}: the two results must not share memory")


def norm_rotary(who: str, like: torch.Tensor, rotary, q_weight, k_weight, eps, interleaved) -> _lib.NormRotary:
    """``en_norm_rotary`` of the arguments these calls share; ``like``: rows of the head size, type and device they are for."""
    D = like.shape[-1]
    how = _lib.NormRotary(eps=float(eps), interleaved=int(bool(interleaved)))
    for w, n in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w is not None:
            _lib.require_gpu(w, n)
            if w.numel() != D or w.dtype != like.dtype or w.device != like.device:
                raise RuntimeError(f"{who}: {n} must hold size_per_head elements of the rows' dtype on their device")
    if rotary is not None:
        cos, sin = rotary
        for t, n in ((cos, "cos"), (sin, "sin")):
            _lib.require_gpu(t, n)
            if t.dim() != 2 or t.dtype != torch.float32 or t.device != like.device:
                raise RuntimeError(f"{who}: {n} must be a float32 [positions, rotary_dim / 2] tensor on the rows' device")
        if cos.shape != sin.shape or cos.shape[0] < 1 or cos.shape[1] < 1 or 2 * cos.shape[1] > D:
            raise RuntimeError(f"{who}: cos and sin must share a shape and cover at most size_per_head channels")
        how.cos, how.sin, how.table_rows, how.rotary_dim = cos.data_ptr(), sin.data_ptr(), cos.shape[0], 2 * cos.shape[1]
    how.q_weight, how.k_weight = _lib.ptr(q_weight) or None, _lib.ptr(k_weight) or None
    return how


def qk_norm_rotary(q, k, batch_size: int, seq_len_list, rotary=None, *, q_weight=None, k_weight=None, eps: float = 1e-6,
                   interleaved: bool = False, positions: Optional[torch.Tensor] = None, out=None):
    """Queries and keys of packed tokens, normed head by head and rotated, in one pass: ``q`` ``[T,Hq,D]`` and ``k`` ``[T,Hk,D]`` are
    views (any token and head strides) of the projection output, fp16, bf16 or fp32, heads of up to 256 channels.  ``rotary`` is the
    pair of :func:`rotary_table` (or ``None``), ``q_weight`` / ``k_weight`` ``[D]`` the gains of the RMS norms (``None``: no norm).
    A token's position is its place in its sequence, or ``positions[token]`` (int32); one outside the table makes the rotated
    channels NaN.  Rows behind the last sequence are left as they are (with ``positions`` every row is a token).  Returns new ``(q, k)``,
    or writes into the two tensors ``out`` names, which may be ``q`` and ``k`` themselves.  ``k`` may be ``None``."""
    who = "qk_norm_rotary"
    if out is None and k is not None and (positions is not None or type(seq_len_list) is SeqInfo):
        pair = _lib.front.qk_norm_rotary(q, k, batch_size, seq_len_list, positions, rotary, q_weight, k_weight, eps, interleaved)
        if pair is not None:
            return pair
    _rows(q, "q", who)
    T, Hq, D = q.shape
    tensors = [q]
    if k is not None:
        _rows(k, "k", who)
        if k.shape[0] != T or k.shape[2] != D or k.dtype != q.dtype or k.device != q.device:
            raise RuntimeError(f"{who}: q and k disagree in tokens, size_per_head, dtype or device")
        tensors.append(k)
    tag = _lib.dtype_tag(q, who)
    how = norm_rotary(who, q, rotary, q_weight, k_weight, eps, interleaved)
    if out is None:
        outs = [torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in tensors]
    else:
        outs = [t for t in out if t is not None]
        if len(outs) != len(tensors) or any(_rows(o, "out", who).shape != t.shape or o.dtype != t.dtype or o.device != t.device
                                            for o, t in zip(outs, tensors)):
            raise RuntimeError(f"{who}: out must be a pair of tensors of q's and k's shapes, dtype and device")
        _not_over(who, tensors, outs)
    info = None
    if positions is None:
        info = seq_info(seq_len_list, batch_size, q.device)
        if info.cu_seqlens is None:
            raise RuntimeError(f"{who}: the lengths of packed rows must come with their offsets (build_seq_info)")
        if info.lens.device != q.device:
            raise RuntimeError(f"{who}: the lengths must be on the rows' device")
    else:
        _lib.require_gpu(positions, "positions")
        if positions.numel() != T or positions.dtype != torch.int32 or positions.device != q.device:
            raise RuntimeError(f"{who}: positions must be a contiguous int32 tensor of one position a token on the rows' device")
    if T and Hq:
        strides = []
        for t in tensors + ([] if k is not None else [q]):
            strides += [t.stride(0), t.stride(1)]
        for t in outs + ([] if k is not None else [q]):
            strides += [t.stride(0), t.stride(1)]
        Hk = 0 if k is None else k.shape[1]
        with _lib.device_guard(q):
            _lib.check(_lib.fn.en_qk_norm_rotary(q.data_ptr(), k.data_ptr() if Hk else None, outs[0].data_ptr(), outs[1].data_ptr() if Hk else None,
                                                 None if info is None else info.cu_seqlens.data_ptr(), _lib.ptr(positions) or None,
                                                 int(batch_size), T, Hq, Hk, D, (ctypes.c_int64 * 8)(*strides), ctypes.byref(how),
                                                 tag, _lib.stream_of(q)), who)
    if out is not None:
        return tuple(out)
    return outs[0], (outs[1] if k is not None else None)


def _new_rows(who: str, q, k_new, v_new, B: int, H: int, D: int, dtype, device):
    """Checks of a decode step's rows; (query heads, their strides)."""
    for t, n in ((k_new, "k_new"), (v_new, "v_new")):
        if _rows(t, n, who).shape != (B, H, D) or t.dtype != dtype or t.device != device:
            raise RuntimeError(f"{who}: {n} must be [B,H,D] of the cache's dtype on its device")
    if q is None:
        return 0, (0, 0)
    if _rows(q, "q", who).shape[0] != B or q.shape[2] != D or q.shape[1] < 1 or q.dtype != dtype or q.device != device:
        raise RuntimeError(f"{who}: q must be [B,Hq,D] of the cache's dtype on its device")
    return q.shape[1], (q.stride(0), q.stride(1))


def kv_pages_append_rotary(q, k_new, v_new, k_pool, v_pool, kv_len_list, page_table, rotary=None, *, q_weight=None, k_weight=None,
                           eps: float = 1e-6, interleaved: bool = False, overflow: Optional[torch.Tensor] = None):
    """``kv_pages_append`` with norms and rotation on the way (see :func:`qk_norm_rotary`), at position ``kv_len[b]``: the new keys go into
    their pages normed and rotated, the values as they are, and the normed, rotated queries ``[B,Hq,D]`` are returned (``Hq`` may
    be any number).  All operands may be strided views of one projection.  A sequence without a page for its next position is handled as there."""
    who = "kv_pages_append_rotary"
    if type(kv_len_list) is SeqInfo:
        turned = _lib.front.kv_pages_append_rotary(q, k_new, v_new, k_pool, v_pool, kv_len_list, page_table, rotary, q_weight, k_weight, eps,
                                                   interleaved, overflow)
        if turned is not None:
            return turned
    ps = _pool(k_pool, "k_pool")
    if _pool(v_pool, "v_pool") != ps or k_pool.shape != v_pool.shape or k_pool.dtype != v_pool.dtype or k_pool.device != v_pool.device:
        raise RuntimeError(f"{who}: K and V must share shapes, strides, dtype and device")
    N, H, P, D = k_pool.shape
    _rows(q, "q", who)
    B = q.shape[0]
    Hq, qs = _new_rows(who, q, k_new, v_new, B, H, D, k_pool.dtype, k_pool.device)
    tag = _lib.dtype_tag(k_pool, who)
    how = norm_rotary(who, q, rotary, q_weight, k_weight, eps, interleaved)
    max_pages = _page_table(page_table, B, who)
    _overflow(overflow, who)
    info = seq_info(kv_len_list, B, k_pool.device)
    for t in (page_table, info.lens) + (() if overflow is None else (overflow,)):
        if t.device != k_pool.device:
            raise RuntimeError(f"{who}: page_table, lengths and overflow must be on the pools' device")
    q_out = torch.empty((B, Hq, D), dtype=q.dtype, device=q.device)
    with _lib.device_guard(k_pool):
        _lib.check(_lib.fn.en_kv_append_paged_rotary(
            q.data_ptr(), k_new.data_ptr(), v_new.data_ptr(), q_out.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(),
            info.lens.data_ptr(), page_table.data_ptr(), B, Hq, H, max_pages, P, N, D,
            (ctypes.c_int64 * 6)(*qs, k_new.stride(0), k_new.stride(1), v_new.stride(0), v_new.stride(1)), (ctypes.c_int64 * 3)(*ps),
            ctypes.byref(how), tag, _lib.ptr(overflow) or None, _lib.stream_of(k_pool)), who)
    return q_out
