"""Decode steps of several drafted tokens a sequence over a paged cache: their attention, which of them are accepted, and the accepted
rows' way into the cache.

The nodes of a step are packed rows: each sequence's newest token, which is certain, as node 0, and behind it the tokens that were drafted,
as a tree of up to 64 nodes whose parents come before their children.  One pass over weights and cache checks them all: project the
nodes, ``decode_attn_tree`` them over the cache and over one another, ``accept_drafts`` from their logits, and
``kv_pages_extend`` the cache, layer by layer, by the accepted nodes' rows.  Only then do lengths advance (``lens.add_(counts)``); nodes that are
not accepted never reach the cache.  No call reads the device, and all can be captured.  The reference decodes one token a step
(energonai/model/attention.py:61-71).
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from .. import _lib
from ..seqinfo import SeqInfo, seq_info
from .attention import _overflow, _page_table, _pool

DRAFT_MAX_NODES = 64
_TYPES = (torch.float16, torch.bfloat16)


class DraftTree(NamedTuple):
    """The trees of a batch.  ``masks`` may be others than ``draft_tree`` makes: bit i of a node's mask says that it sees node i."""
    parents: torch.Tensor       # int32 [nodes]: a node's parent in its sequence, -1 for none
    masks: torch.Tensor         # int64 [nodes]: the nodes on the way from the root, the node among them
    depths: torch.Tensor        # int32 [nodes]: steps from the root; kv_len + depth is the node's position
    info: SeqInfo               # the sequences' numbers of nodes, with their offsets
    max_nodes: int              # at least the largest of them, at most 64


def draft_tree(parents, node_counts, batch_size: int, max_nodes: int = DRAFT_MAX_NODES) -> DraftTree:
    """Masks and depths of the nodes of ``batch_size`` trees.  ``parents`` is int32 ``[nodes]``, sequence by sequence; a number that is not
    that of an earlier node of the sequence counts as -1.  ``node_counts``: int32 or int64 numbers, a list, or a ``SeqInfo`` of them.
    Nodes past the 64th of a sequence do not exist for any call, nor do those past ``max_nodes`` for the calls that take the tree; their rows, and
    rows behind the last sequence, have mask and depth 0."""
    who = "draft_tree"
    _lib.require_gpu(parents, "parents")
    if parents.dim() != 1 or parents.dtype != torch.int32:
        raise RuntimeError(f"{who}: parents must be an int32 [nodes] tensor")
    if not 1 <= int(max_nodes) <= DRAFT_MAX_NODES:
        raise RuntimeError(f"{who}: max_nodes must be 1 .. {DRAFT_MAX_NODES}")
    info = _offsets(who, node_counts, int(batch_size), parents.device)
    new = torch.empty if int(batch_size) > 0 else torch.zeros            # no sequence, no launch
    masks, depths = (new(parents.shape, dtype=t, device=parents.device) for t in (torch.int64, torch.int32))
    with _lib.device_guard(parents):
        _lib.check(_lib.fn.en_draft_tree(parents.data_ptr(), info.cu_seqlens.data_ptr(), int(batch_size), parents.numel(), masks.data_ptr(),
                                         depths.data_ptr(), _lib.stream_of(parents)), who)
    return DraftTree(parents, masks, depths, info, int(max_nodes))


def _offsets(who: str, counts, batch: int, device) -> SeqInfo:
    info = seq_info(counts, batch, device)
    if info.cu_seqlens is None or info.lens.device != device:
        raise RuntimeError(f"{who}: the numbers of nodes must come with their offsets (build_seq_info), on the device of the nodes")
    return info


def _tree(who: str, tree, device, nodes: int, batch: int, *fields: str) -> SeqInfo:
    """Checks the tensors ``fields`` of a tree against the rows of a call; its offsets."""
    if not isinstance(tree, DraftTree):
        raise RuntimeError(f"{who}: tree must be a DraftTree")
    for n in fields:
        t = getattr(tree, n)
        _lib.require_gpu(t, n)
        if t.dim() != 1 or t.numel() != nodes or t.dtype != (torch.int64 if n == "masks" else torch.int32) or t.device != device:
            raise RuntimeError(f"{who}: the tree's {n} must be one for each of the {nodes} nodes, on their device")
    if not 1 <= int(tree.max_nodes) <= DRAFT_MAX_NODES:
        raise RuntimeError(f"{who}: max_nodes must be 1 .. {DRAFT_MAX_NODES}")
    return _offsets(who, tree.info, batch, device)


def _kv_pages(who: str, k_pool, v_pool, page_table, batch: int) -> _lib.KvPages:
    ks, vs = _pool(k_pool, "k_pool"), _pool(v_pool, "v_pool")
    if v_pool.shape != k_pool.shape or v_pool.dtype != k_pool.dtype or v_pool.device != k_pool.device:
        raise RuntimeError(f"{who}: k_pool and v_pool must share shape, dtype and device")
    N, H, P, D = k_pool.shape
    pages = _page_table(page_table, batch, who)
    if page_table.device != k_pool.device:
        raise RuntimeError(f"{who}: page_table must be on the pools' device")
    c = _lib.KvPages(k_pool.data_ptr(), v_pool.data_ptr(), page_table.data_ptr())
    one = lambda s: [s[0] if N > 1 else 0, s[1] if H > 1 else 0, s[2]]  # noqa: E731
    c.strides[:] = one(ks) + one(vs)
    c.num_pages, c.page_size, c.max_pages_per_seq, c.batch, c.head_num, c.size_per_head = N, P, pages, batch, H, D
    c.dtype = _lib.dtype_tag(k_pool, who)
    return c


def _node_rows(who: str, t, name: str, nodes: Optional[int], heads: Optional[int], D: int, pool) -> torch.Tensor:
    _lib.require_gpu(t, name, contiguous=False)
    if t.dim() != 3 or t.shape[2] != D or (heads is not None and t.shape[1] != heads) or (nodes is not None and t.shape[0] != nodes) \
            or t.dtype != pool.dtype or t.device != pool.device:
        raise RuntimeError(f"{who}: {name} must be [nodes, heads, {D}] of the pools' dtype on their device")
    return t


def _vectors(t):
    """``t``, or a copy where its rows do not lie as 16-byte vectors."""
    ok = t.stride(2) == 1 and t.stride(0) % 8 == 0 and t.stride(1) % 8 == 0 and t.data_ptr() % 16 == 0
    if ok:
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _apart(a, b) -> bool:
    """Whether two tensors, any strides of at least 0, share no memory."""
    def ends(t):
        last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
        return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()
    if a.numel() == 0 or b.numel() == 0:
        return True
    (a0, a1), (b0, b1) = ends(a), ends(b)
    return a1 <= b0 or b1 <= a0


def decode_attn_tree_workspace_bytes(batch_size: int, q_heads: int, head_num: int, capacity: int, size_per_head: int, max_nodes: int) -> int:
    """Bytes of the buffer through which ``decode_attn_tree`` passes its partial results (0: it needs none for caches of this
    capacity, in positions a sequence)."""
    return int(_lib.fn.en_decode_attn_tree_workspace_bytes(int(batch_size), int(q_heads), int(head_num), int(capacity), int(size_per_head),
                                                           int(max_nodes)))


def decode_attn_tree(q, k_new, v_new, k_pool, v_pool, kv_len_list, page_table, tree, *, scale: Optional[float] = None,
                     out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None):
    """``decode_attn_paged`` of several nodes a sequence: ``q`` is ``[nodes, Hq, D]``, ``k_new`` and ``v_new`` ``[nodes, H, D]``, packed, with
    ``Hq`` a multiple of the pools' heads (neighbouring query heads share a key head).  A node sees its sequence's ``kv_len`` cached positions
    and those of its sequence's nodes that its mask names.  Returns ``[nodes, Hq, D]``: zeros where a node sees nothing; rows of nodes
    that do not exist are left as they are.  fp16 and bf16, heads of a multiple of 8 channels up to 128.  ``scale`` defaults to ``D ** -0.5``;
    ``out`` may be ``q``; ``workspace``: any tensor of ``decode_attn_tree_workspace_bytes`` bytes (``None``: a temporary)."""
    who = "decode_attn_tree"
    if out is None and workspace is None and type(tree) is DraftTree:
        ctx = _lib.front.decode_attn_tree(q, k_new, v_new, k_pool, v_pool, kv_len_list, page_table, tree, scale)
        if ctx is not None:
            return ctx
    B = page_table.shape[0] if isinstance(page_table, torch.Tensor) and page_table.dim() == 2 else 0
    c = _kv_pages(who, k_pool, v_pool, page_table, B)
    if k_pool.dtype not in _TYPES:
        raise RuntimeError(f"{who}: Datatype not implemented ({k_pool.dtype}); expected float16 or bfloat16")
    H, D, device = c.head_num, c.size_per_head, k_pool.device
    T, Hq = _node_rows(who, q, "q", None, None, D, k_pool).shape[:2]
    if H < 1 or Hq < H or Hq % H:
        raise RuntimeError(f"{who}: q must have a multiple of the pools' {H} heads")
    for t, n in ((k_new, "k_new"), (v_new, "v_new")):
        _node_rows(who, t, n, T, H, D, k_pool)
    if any(not p.data_ptr() % 16 == 0 or any(s % 8 for s, n in zip(p.stride()[:3], p.shape) if n > 1) for p in (k_pool, v_pool)):
        raise RuntimeError(f"{who}: the pools' rows must lie as 16-byte vectors")
    info = _tree(who, tree, device, T, B, "masks")
    lens = _lens(who, kv_len_list, B, device)
    q_, k_, v_ = _vectors(q), _vectors(k_new), _vectors(v_new)
    if out is None:
        out = torch.empty((T, Hq, D), dtype=q.dtype, device=device)
    else:
        _lib.require_gpu(out, "out")
        same = out.data_ptr() == q_.data_ptr() and q_.is_contiguous()
        if out.shape != (T, Hq, D) or out.dtype != q.dtype or out.device != device or out.data_ptr() % 16 \
                or not (same or _apart(out, q_)) or not all(_apart(out, t) for t in (k_, v_, k_pool, v_pool)):
            raise RuntimeError(f"{who}: out must be a contiguous [nodes, Hq, D] tensor of q's dtype on its device, q itself or apart from the operands")
    need = decode_attn_tree_workspace_bytes(B, Hq, H, c.max_pages_per_seq * c.page_size, D, tree.max_nodes)
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
    _lib.require_gpu(workspace, "workspace")
    if workspace.device != device or workspace.numel() * workspace.element_size() < need:
        raise RuntimeError(f"{who}: workspace must hold {need} bytes on the pools' device")
    scale = float(D) ** -0.5 if scale is None else float(scale)
    with _lib.device_guard(q):
        _lib.check(_lib.fn.en_decode_attn_tree(q_.data_ptr(), k_.data_ptr(), v_.data_ptr(), _token_head(q_, k_, v_), out.data_ptr(), ctypes.byref(c),
                                               lens.lens.data_ptr(), info.cu_seqlens.data_ptr(), tree.masks.data_ptr(), T, tree.max_nodes, Hq, scale,
                                               _lib.ptr(workspace) or None, workspace.numel() * workspace.element_size(), _lib.stream_of(q)), who)
    return out


def _token_head(*rows):
    """(token, head) strides; those of a dimension of one may be any."""
    return (ctypes.c_int64 * (2 * len(rows)))(*[t.stride(d) if t.shape[d] > 1 else 0 for t in rows for d in (0, 1)])


def _lens(who: str, lens, B: int, device) -> SeqInfo:
    info = seq_info(lens, B, device)
    if info.lens.device != device:
        raise RuntimeError(f"{who}: the lengths must be on the pools' device")
    return info


def accept_drafts(logits, tokens, tree):
    """Which nodes a greedy decoding would have chosen: from node 0, which is certain, on, the lowest child whose token has the largest of
    the node's logits (the lowest index of equal ones; NaN counts as the largest), until there is none.  ``logits`` ``[nodes, vocab]``
    with contiguous rows, ``tokens`` int32 or int64 ``[nodes]``.  Returns ``(path, counts, next_tokens)``: int32 ``[B, max_nodes]``, the
    accepted nodes and -1 behind them; int32 ``[B]``, how many (at least 1; 0 for a sequence without nodes); int64 ``[B]``, the token that follows (-1).

    It is exact for the logits that it is given.  A model's logits of a node differ, within its operators' roundings, from those that a step of single tokens gives:
    sums go in another order and, with weights in 4 bits, more than 64 rows are multiplied by rounded weights.  Where a row's two largest logits are nearer than
    that, the two ways of decoding may choose differently."""
    who = "accept_drafts"
    if type(tree) is DraftTree:
        found = _lib.front.accept_drafts(logits, tokens, tree)
        if found is not None:
            return found
    _lib.require_gpu(logits, "logits", contiguous=False)
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1) or logits.shape[1] < 1:
        raise RuntimeError(f"{who}: logits must be a [nodes, vocab] tensor with contiguous rows")
    T, V = logits.shape
    dtype = _lib.dtype_tag(logits, who)
    _lib.require_gpu(tokens, "tokens")
    if tokens.shape != (T,) or tokens.dtype not in (torch.int32, torch.int64) or tokens.device != logits.device:
        raise RuntimeError(f"{who}: tokens must be int32 or int64, one for each of the logits' {T} rows, on their device")
    if not isinstance(tree, DraftTree):
        raise RuntimeError(f"{who}: tree must be a DraftTree")
    B = tree.info.batch_size
    info = _tree(who, tree, logits.device, T, B, "parents")
    path = torch.empty((B, tree.max_nodes), dtype=torch.int32, device=logits.device)
    counts = torch.empty(B, dtype=torch.int32, device=logits.device)
    following = torch.empty(B, dtype=torch.int64, device=logits.device)
    need = int(_lib.fn.en_accept_drafts_workspace_bytes(T, V, dtype))
    workspace = torch.empty(need, dtype=torch.uint8, device=logits.device)
    with _lib.device_guard(logits):
        _lib.check(_lib.fn.en_accept_drafts(logits.data_ptr(), logits.stride(0) if T > 1 else V, V, tokens.data_ptr(), int(tokens.dtype == torch.int64),
                                            tree.parents.data_ptr(), info.cu_seqlens.data_ptr(), B, T, tree.max_nodes, path.data_ptr(),
                                            counts.data_ptr(), following.data_ptr(), dtype, _lib.ptr(workspace) or None, need, _lib.stream_of(logits)), who)
    return path, counts, following


def kv_pages_extend(k_new, v_new, k_pool, v_pool, kv_len_list, page_table, tree, path, counts, *, overflow: Optional[torch.Tensor] = None) -> None:
    """``kv_pages_append`` of the accepted nodes: the rows of nodes ``path[b, i]``, ``i < counts[b]``, of ``k_new`` and ``v_new`` ``[nodes, H, D]``
    (any token and head strides) become positions ``kv_len[b] + i`` of sequence ``b``.  The caller advances the lengths afterwards.  Entries of
    ``path`` that name no node of the tree are passed over; a position that has no page in the pool is not written and counted in ``overflow``.  Up to 65535
    sequences."""
    who = "kv_pages_extend"
    if type(tree) is DraftTree and _lib.front.kv_pages_extend(k_new, v_new, k_pool, v_pool, kv_len_list, page_table, tree, path, counts, overflow):
        return
    B = page_table.shape[0] if isinstance(page_table, torch.Tensor) and page_table.dim() == 2 else 0
    c = _kv_pages(who, k_pool, v_pool, page_table, B)
    T = k_new.shape[0] if isinstance(k_new, torch.Tensor) and k_new.dim() == 3 else 0
    for t, n in ((k_new, "k_new"), (v_new, "v_new")):
        if _node_rows(who, t, n, T, c.head_num, c.size_per_head, k_pool).stride(2) != 1 and c.size_per_head > 1:
            raise RuntimeError(f"{who}: {n} must have contiguous channels")
    if not isinstance(tree, DraftTree):
        raise RuntimeError(f"{who}: tree must be a DraftTree")
    info = _tree(who, tree, k_pool.device, T, B)
    for t, n, shape in ((path, "path", (B, path.shape[1] if isinstance(path, torch.Tensor) and path.dim() == 2 else 0)), (counts, "counts", (B,))):
        _lib.require_gpu(t, n)
        if t.shape != shape or t.dtype != torch.int32 or t.device != k_pool.device:
            raise RuntimeError(f"{who}: path must be int32 [batch, steps] and counts int32 [batch], on the pools' device")
    _overflow(overflow, who)
    if overflow is not None and overflow.device != k_pool.device:
        raise RuntimeError(f"{who}: overflow must be on the pools' device")
    lens = _lens(who, kv_len_list, B, k_pool.device)
    with _lib.device_guard(k_pool):
        _lib.check(_lib.fn.en_kv_extend_paged_nodes(k_new.data_ptr(), v_new.data_ptr(), _token_head(k_new, v_new), ctypes.byref(c), lens.lens.data_ptr(),
                                                    info.cu_seqlens.data_ptr(), T, tree.max_nodes, path.data_ptr(), path.shape[1], counts.data_ptr(),
                                                    _lib.ptr(overflow) or None, _lib.stream_of(k_pool)), who)
