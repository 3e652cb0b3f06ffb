"""A paged K/V cache in 8 bits, and the decode attention that reads it.

The positions of a sequence are taken in blocks of 16.  A full block lies in a page as codes, int8 or float8_e4m3fn, with one float32 scale for
the block and head of its keys and one of its values: with a the block's largest magnitude and M the largest code (127; 448)
``scale = a / M`` and ``code = round(x * (M / a))``, computed in fp32 and rounded to nearest even (a < 2^-100: zeros; a value that is
not finite: the scale is NaN).  The positions behind the last full block stay in 16 bits in a tail of the sequence, so that every block is
quantized once, from full values, and a cache filled by a prompt is the one that appending its positions gives.  The reference keeps its
history in the projection's type (energonai/model/attention.py:61-71).

Heads of 16, 32, .. 128 channels, fp16 and bf16, pages of a power of two of at least 16 positions.  A page id outside the pool reads as
zeros and is not written, nor is the tail of positions that would lie there.  A new row that is lost for want of a page stays lost: named later,
the page has whatever it (or, in an unfinished block, the tail) held in that position.

A tail belongs to its sequence's place in the batch, as the row of ``page_table`` does, and holds the positions behind the last full block
alone: a sequence that moves to another place takes both along, and a length may go back to no less than the last multiple of 16 it has
passed (shorter: the sequence is filled again, for instance from ``kv8_pages_read``).
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from .. import _lib
from ..seqinfo import SeqInfo, seq_info
from .attention import _overflow
from .rotary import _new_rows, _rows, norm_rotary

KV8_BLOCK = 16
_CODES = {torch.int8: 0, torch.float8_e4m3fn: 1}
_TYPES = (torch.float16, torch.bfloat16)


class KV8Pages(NamedTuple):
    """The tensors of a cache; the calls of this module take any tuple of them.  Page and head strides are free for pools and scales."""
    k_pages: torch.Tensor       # [pages, H, P, D] codes
    v_pages: torch.Tensor       # [pages, H, P / 16, D, 16] codes of the same type: a block's positions lie innermost
    k_scales: torch.Tensor      # [pages, H, P / 16] float32
    v_scales: torch.Tensor
    k_tail: torch.Tensor        # [B, H, 16, D] fp16 or bf16
    v_tail: torch.Tensor        # [B, H, D, 16]
    page_table: torch.Tensor    # int32 [B, max_pages_per_seq]


def kv8_pages(pool_pages: int, batch_size: int, head_num: int, page_size: int, size_per_head: int, max_pages_per_seq: int, dtype, device,
              code_dtype=torch.int8) -> KV8Pages:
    """A new cache: zeros, and a table that names no page."""
    if code_dtype not in _CODES or dtype not in _TYPES:
        raise RuntimeError("kv8_pages: Datatype not implemented; expected codes in int8 or float8_e4m3fn and float16 or bfloat16 rows")
    if page_size < KV8_BLOCK or page_size & (page_size - 1) or size_per_head % 16 or not 16 <= size_per_head <= 128:
        raise RuntimeError("kv8_pages: pages of a power of two of at least 16 positions, heads of 16, 32, .. 128 channels")
    zeros = lambda shape, t: torch.zeros(shape, dtype=t, device=device)  # noqa: E731
    blocks = page_size // KV8_BLOCK
    codes = lambda shape: zeros(shape, torch.int8).view(code_dtype)  # noqa: E731
    return KV8Pages(codes((pool_pages, head_num, page_size, size_per_head)), codes((pool_pages, head_num, blocks, size_per_head, KV8_BLOCK)),
                    zeros((pool_pages, head_num, blocks), torch.float32), zeros((pool_pages, head_num, blocks), torch.float32),
                    zeros((batch_size, head_num, KV8_BLOCK, size_per_head), dtype), zeros((batch_size, head_num, size_per_head, KV8_BLOCK), dtype),
                    torch.full((batch_size, max_pages_per_seq), -1, dtype=torch.int32, device=device))


def _cache(cache, who: str) -> _lib.Kv8Cache:
    """``en_kv8_cache`` of a cache's tensors."""
    if len(cache) != 7:
        raise RuntimeError(f"{who}: cache must be the seven tensors of KV8Pages")
    kp, vp, ks, vs, kt, vt, table = cache
    names = KV8Pages._fields
    for t, n in zip(cache, names):
        _lib.require_gpu(t, n, contiguous=n in ("k_tail", "v_tail", "page_table"))
        if t.device != kp.device:
            raise RuntimeError(f"{who}: the cache's tensors must be on one device")
    if kp.dtype not in _CODES or vp.dtype != kp.dtype or kt.dtype not in _TYPES or vt.dtype != kt.dtype or ks.dtype != torch.float32 \
            or vs.dtype != torch.float32 or table.dtype != torch.int32:
        raise RuntimeError(f"{who}: Datatype not implemented; expected codes in int8 or float8_e4m3fn, float32 scales, float16 or bfloat16 "
                           f"tails and an int32 page_table")
    if kp.dim() != 4 or kt.dim() != 4 or table.dim() != 2:
        raise RuntimeError(f"{who}: k_pages must be [pages, H, P, D], k_tail [B, H, 16, D] and page_table [B, max_pages_per_seq]")
    N, H, P, D = kp.shape
    B, blocks = table.shape[0], P // KV8_BLOCK
    if N < 1 or P < KV8_BLOCK or P & (P - 1) or D % 16 or not 16 <= D <= 128:
        raise RuntimeError(f"{who}: a pool of at least one page, pages of a power of two of at least 16 positions, heads of 16, 32, .. 128 channels")
    if vp.shape != (N, H, blocks, D, KV8_BLOCK) or ks.shape != (N, H, blocks) or vs.shape != ks.shape or kt.shape != (B, H, KV8_BLOCK, D) \
            or vt.shape != (B, H, D, KV8_BLOCK):
        raise RuntimeError(f"{who}: v_pages must be [pages, H, P / 16, D, 16], scales [pages, H, P / 16], tails [B, H, 16, D] and [B, H, D, 16]")
    if kp.stride()[2:] != (D, 1) or vp.stride()[3:] != (KV8_BLOCK, 1) or (blocks > 1 and (vp.stride(2), ks.stride(2), vs.stride(2)) != (D * KV8_BLOCK, 1, 1)):
        raise RuntimeError(f"{who}: the positions of a page and head must be contiguous in pools and scales")
    c = _lib.Kv8Cache(kp.data_ptr(), vp.data_ptr(), ks.data_ptr(), vs.data_ptr(), kt.data_ptr(), vt.data_ptr(), table.data_ptr())
    strides = lambda t: [t.stride(0) if N > 1 else 0, t.stride(1) if H > 1 else 0]  # noqa: E731
    c.code_strides[:], c.scale_strides[:] = strides(kp) + strides(vp), strides(ks) + strides(vs)
    c.num_pages, c.page_size, c.max_pages_per_seq, c.batch, c.head_num, c.size_per_head = N, P, table.shape[1], B, H, D
    c.code, c.dtype = _CODES[kp.dtype], _lib.dtype_tag(kt, who)
    return c


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two contiguous tensors of a device share memory."""
    return a.data_ptr() < b.data_ptr() + b.numel() * b.element_size() and b.data_ptr() < a.data_ptr() + a.numel() * a.element_size()


def _lens(who: str, lens, B: int, device):
    info = seq_info(lens, B, device)
    if info.lens.device != device:
        raise RuntimeError(f"{who}: the lengths must be on the cache's device")
    return info


def kv8_pages_fill(k_src, v_src, cache, batch_size: int, max_seq_len: int, seq_len_list, *, overflow: Optional[torch.Tensor] = None) -> None:
    """Prefill: rows ``cu[b] + s`` of ``k_src`` / ``v_src`` (``[T,H,D]`` views, any token and head strides) become the positions
    ``s < min(len[b], max_seq_len)`` of sequence ``b``: full blocks into the pages that ``page_table`` names, the rest into the tails.  Positions whose
    page id lies outside the pool are not written and counted in ``overflow``."""
    who = "kv8_pages_fill"
    if type(seq_len_list) is SeqInfo and _lib.front.kv8_pages_fill(k_src, v_src, cache, batch_size, max_seq_len, seq_len_list, overflow):
        return
    c = _cache(cache, who)
    kt, device = cache[4], cache[4].device
    for t, n in ((k_src, "k_src"), (v_src, "v_src")):
        if _rows(t, n, who).shape[1:] != (c.head_num, c.size_per_head) or t.dtype != kt.dtype or t.device != device:
            raise RuntimeError(f"{who}: {n} must be [T,H,D] of the tails' dtype on the cache's device")
    if k_src.shape[0] != v_src.shape[0] or int(batch_size) != c.batch or int(max_seq_len) < 0:
        raise RuntimeError(f"{who}: K and V must have the same tokens, and batch_size must be the cache's")
    _overflow(overflow, who)
    if overflow is not None and overflow.device != device:
        raise RuntimeError(f"{who}: overflow must be on the cache's device")
    info = _lens(who, seq_len_list, c.batch, device)
    if info.cu_seqlens is None:
        raise RuntimeError(f"{who}: the lengths of packed rows must come with their offsets (build_seq_info)")
    if k_src.shape[0] == 0:
        return
    with _lib.device_guard(kt):
        _lib.check(_lib.fn.en_kv8_fill(k_src.data_ptr(), v_src.data_ptr(), ctypes.byref(c), info.cu_seqlens.data_ptr(), k_src.shape[0], int(max_seq_len),
                                       (ctypes.c_int64 * 4)(k_src.stride(0), k_src.stride(1), v_src.stride(0), v_src.stride(1)),
                                       _lib.ptr(overflow) or None, _lib.stream_of(kt)), who)


def kv8_pages_append(q, k_new, v_new, cache, kv_len_list, rotary=None, *, q_weight=None, k_weight=None, eps: float = 1e-6,
                     interleaved: bool = False, overflow: Optional[torch.Tensor] = None):
    """``kv_pages_append_rotary`` into a cache in 8 bits: the new rows of position ``kv_len[b]`` go into the tails, and a block that they
    complete into its page.  Returns the normed, rotated queries (``q`` may be ``None``: then nothing).  The caller advances the lengths
    afterwards.  A sequence whose position has no page keeps its cache, loses the new rows and is counted in ``overflow``."""
    who = "kv8_pages_append"
    if q is not None and type(kv_len_list) is SeqInfo:
        turned = _lib.front.kv8_pages_append(q, k_new, v_new, cache, kv_len_list, rotary, q_weight, k_weight, eps, interleaved, overflow)
        if turned is not None:
            return turned
    c = _cache(cache, who)
    kt, device = cache[4], cache[4].device
    Hq, qs = _new_rows(who, q, k_new, v_new, c.batch, c.head_num, c.size_per_head, kt.dtype, device)
    how = norm_rotary(who, k_new, rotary, q_weight, k_weight, eps, interleaved)
    _overflow(overflow, who)
    if overflow is not None and overflow.device != device:
        raise RuntimeError(f"{who}: overflow must be on the cache's device")
    info = _lens(who, kv_len_list, c.batch, device)
    q_out = None if q is None else torch.empty((c.batch, Hq, c.size_per_head), dtype=q.dtype, device=device)
    with _lib.device_guard(kt):
        _lib.check(_lib.fn.en_kv8_append(_lib.ptr(q) or None, k_new.data_ptr(), v_new.data_ptr(), _lib.ptr(q_out) or None, ctypes.byref(c),
                                         info.lens.data_ptr(), Hq,
                                         (ctypes.c_int64 * 6)(*qs, k_new.stride(0), k_new.stride(1), v_new.stride(0), v_new.stride(1)),
                                         ctypes.byref(how), _lib.ptr(overflow) or None, _lib.stream_of(kt)), who)
    return q_out


def kv8_pages_read(cache, kv_len_list, max_seq_len: int, *, first: Optional[torch.Tensor] = None, out=None):
    """The cached positions ``first[b] + s``, ``s < max_seq_len``, as ``(k, v)`` of ``[B,H,max_seq_len,D]`` in the tails' type, zeros from
    ``kv_len[b]`` on: what a prompt that goes on from a cached one attends to, or what a swapped-out sequence keeps.  ``first`` is int32 ``[B]``
    (``None``: 0, as which a negative one counts)."""
    who = "kv8_pages_read"
    if out is None and type(kv_len_list) is SeqInfo:
        pair = _lib.front.kv8_pages_read(cache, kv_len_list, max_seq_len, first)
        if pair is not None:
            return pair
    c = _cache(cache, who)
    kt, device = cache[4], cache[4].device
    info = _lens(who, kv_len_list, c.batch, device)
    S = int(max_seq_len)
    if S < 0:
        raise RuntimeError(f"{who}: max_seq_len must not be negative")
    if first is not None:
        _lib.require_gpu(first, "first")
        if first.numel() != c.batch or first.dtype != torch.int32 or first.device != device:
            raise RuntimeError(f"{who}: first must be a contiguous int32 [batch] tensor on the cache's device")
    shape = (c.batch, c.head_num, S, c.size_per_head)
    if out is None:
        out = (torch.empty(shape, dtype=kt.dtype, device=device), torch.empty(shape, dtype=kt.dtype, device=device))
    else:
        for t in out:
            _lib.require_gpu(t, "out")
        if len(out) != 2 or any(t.shape != shape or t.dtype != kt.dtype or t.device != device for t in out) or _overlap(*out):
            raise RuntimeError(f"{who}: out must be two contiguous [B,H,max_seq_len,D] tensors of the tails' dtype on the cache's device, apart from one another")
    with _lib.device_guard(kt):
        _lib.check(_lib.fn.en_kv8_read(ctypes.byref(c), info.lens.data_ptr(), _lib.ptr(first) or None, S, out[0].data_ptr(), out[1].data_ptr(),
                                       _lib.stream_of(kt)), who)
    return tuple(out)


def decode_attn_kv8_workspace_bytes(batch_size: int, q_heads: int, head_num: int, capacity: int, size_per_head: int) -> int:
    """Bytes of the buffer through which ``decode_attn_kv8`` passes its partial results (0: caches of this capacity, in positions a
    sequence, need none)."""
    return int(_lib.fn.en_decode_attn_kv8_workspace_bytes(int(batch_size), int(q_heads), int(head_num), int(capacity), int(size_per_head)))


def decode_attn_kv8(q, cache, kv_len_list, *, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                    workspace: Optional[torch.Tensor] = None):
    """``decode_attn_paged`` over a cache in 8 bits: ``q`` is ``[B,Hq,1,D]`` (or ``[B,Hq,D]``) with ``Hq`` a multiple of the cache's heads,
    neighbouring query heads sharing a key head; ``[B,Hq,1,D]``, zeros for an empty sequence.  ``scale`` defaults to
    ``size_per_head ** -0.5``.  ``workspace``: any tensor of ``decode_attn_kv8_workspace_bytes`` bytes (``None``: a temporary)."""
    who = "decode_attn_kv8"
    if out is None and workspace is None and type(kv_len_list) is SeqInfo:
        ctx = _lib.front.decode_attn_kv8(q, cache, kv_len_list, scale)
        if ctx is not None:
            return ctx
    c = _cache(cache, who)
    device = cache[4].device
    _lib.require_gpu(q, "q", contiguous=False)
    row = c.batch * c.head_num * c.size_per_head
    if q.dim() < 3 or q.shape[0] != c.batch or q.shape[-1] != c.size_per_head or q.dtype != cache[4].dtype or q.device != device \
            or q.numel() != c.batch * q.shape[1] * c.size_per_head or (row and q.numel() % row) or q.shape[1] < c.head_num:
        raise RuntimeError(f"{who}: q must be [B,Hq,1,D] of the tails' dtype on the cache's device, Hq a multiple of the cache's heads")
    B, Hq, D = c.batch, q.shape[1], c.size_per_head
    q_ = q.reshape(B, Hq, D).contiguous()
    if q_.data_ptr() % 16:
        q_ = q_.clone()
    info = _lens(who, kv_len_list, B, device)
    if out is None:
        out = torch.empty((B, Hq, 1, D), dtype=q.dtype, device=device)
    else:
        _lib.require_gpu(out, "out")
        if out.numel() != B * Hq * D or out.dtype != q.dtype or out.device != device or (out.data_ptr() != q_.data_ptr() and _overlap(out, q_)):
            raise RuntimeError(f"{who}: out must be a contiguous [B,Hq,1,D] tensor of q's dtype on its device, q itself or apart from it")
    need = decode_attn_kv8_workspace_bytes(B, Hq, c.head_num, c.max_pages_per_seq * c.page_size, D)
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
    _lib.require_gpu(workspace, "workspace")
    if workspace.device != device or workspace.numel() * workspace.element_size() < need:
        raise RuntimeError(f"{who}: workspace must hold {need} bytes on the cache's device")
    scale = float(D) ** -0.5 if scale is None else float(scale)
    with _lib.device_guard(q):
        _lib.check(_lib.fn.en_decode_attn_kv8(q_.data_ptr(), out.data_ptr(), ctypes.byref(c), info.lens.data_ptr(), Hq, scale,
                                              _lib.ptr(workspace) or None, workspace.numel() * workspace.element_size(), _lib.stream_of(q)), who)
    return out
