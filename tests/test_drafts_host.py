"""What the entry points of drafted steps and 4-bit weights refuse before anything reaches the device, and the plain restatement that the GPU
tests compare with."""
import ctypes
import os
import re

import pytest
import torch

from oracle import drafts as ref

NULL, SHAPE, DTYPE, ALIGN, UNSUPPORTED = -1, -2, -3, -4, -5
PTR = 1 << 20                                             # an address that nothing reads: every call here ends in a refusal or has nothing to do


def _lib():
    from energonai_amd import _lib as lib
    return lib


def _pages(**kw):
    c = _lib().KvPages(PTR, PTR, PTR)
    c.strides[:] = [4096, 2048, 64] * 2
    for n, v in {**dict(num_pages=4, page_size=32, max_pages_per_seq=2, batch=3, head_num=2, size_per_head=64, dtype=1), **kw}.items():
        if n == "strides":
            c.strides[:] = v
        else:
            setattr(c, n, v)
    return c


def test_structures_match_the_header():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(root, "include", "energon_hip.h")).read(), flags=re.S)
    for struct, cls in (("en_kv_pages", _lib().KvPages), ("en_w4_weight", _lib().W4)):
        body = re.search(r"typedef struct %s \{(.*?)\}" % struct, text, flags=re.S).group(1)
        names = [re.sub(r"[\s*]|\[.*\]", "", n) for line in body.split(";") if line.strip() for n in re.sub(r"^\s*(const\s+)?\w+\s", "", line.strip()).split(",")]
        assert names == [f[0] for f in cls._fields_], struct


def test_tree_refuses():
    fn = _lib().fn.en_draft_tree
    assert fn(PTR, PTR, 0, 4, PTR, PTR, None) == 0 and fn(PTR, PTR, 1, 0, PTR, PTR, None) == 0
    assert fn(PTR, PTR, -1, 4, PTR, PTR, None) == SHAPE and fn(PTR, PTR, 1, 1 << 31, PTR, PTR, None) == SHAPE
    for i in (0, 1, 4, 5):
        args = [PTR, PTR, 1, 4, PTR, PTR, None]
        args[i] = None
        assert fn(*args) == NULL
        args[i] = PTR + 2
        assert fn(*args) == ALIGN


def test_attention_refuses():
    fn = _lib().fn.en_decode_attn_tree

    def call(q=PTR, kn=PTR, vn=PTR, st=(1536, 64) * 3, ctx=PTR, lens=PTR, cu=PTR, masks=PTR, nodes=5, max_nodes=4, hq=4, scale=0.125, ws=PTR, ws_bytes=1 << 40, cache=None, **kw):
        c = _pages(**kw) if cache is None else cache
        return fn(q, kn, vn, None if st is None else (ctypes.c_int64 * 6)(*st), ctx, ctypes.byref(c), lens, cu, masks, nodes, max_nodes, hq, scale, ws, ws_bytes, None)
    assert call(nodes=0) == 0 and call(batch=0) == 0
    for kw in (dict(q=None), dict(kn=None), dict(vn=None), dict(st=None), dict(ctx=None), dict(lens=None), dict(cu=None), dict(masks=None)):
        assert call(**kw) == NULL, kw
    for dtype in (0, 3, -1):
        assert call(dtype=dtype) == DTYPE
    for kw in (dict(size_per_head=60), dict(size_per_head=136), dict(scale=0.0), dict(scale=float("nan")), dict(page_size=48), dict(page_size=8)):
        assert call(**kw) == UNSUPPORTED, kw
    for kw in (dict(hq=3), dict(hq=1), dict(max_nodes=65), dict(max_nodes=-1), dict(nodes=-1), dict(nodes=1 << 31), dict(head_num=0), dict(num_pages=0),
               dict(max_pages_per_seq=-1), dict(batch=-1), dict(max_pages_per_seq=1 << 27), dict(strides=[-8, 2048, 64, 4096, 2048, 64])):
        assert call(**kw) == SHAPE, kw
    for kw in (dict(q=PTR + 8), dict(kn=PTR + 2), dict(ctx=PTR + 8), dict(st=(1536, 64, 1540, 64, 1536, 64)), dict(strides=[4096, 2048, 68] + [4096, 2048, 64])):
        assert call(**kw) == ALIGN, kw
    no_pages = _pages()
    no_pages.k_pool = None
    assert call(cache=no_pages) == NULL
    need = _lib().fn.en_decode_attn_tree_workspace_bytes(1, 64, 8, 200000, 128, 64)
    assert need >= 0
    if need:
        long = dict(batch=1, head_num=8, hq=64, max_pages_per_seq=6250, size_per_head=128, max_nodes=64)
        assert call(ws_bytes=need - 1, **long) == SHAPE and call(ws=None, **long) == NULL and call(ws=PTR + 4, **long) == ALIGN


def test_acceptance_refuses():
    fn = _lib().fn.en_accept_drafts

    def call(logits=PTR, stride=100, vocab=100, tokens=PTR, i64=1, parents=PTR, cu=PTR, batch=2, nodes=5, max_nodes=4, path=PTR, counts=PTR, nxt=PTR, dtype=1, ws=PTR, ws_bytes=1 << 30):
        return fn(logits, stride, vocab, tokens, i64, parents, cu, batch, nodes, max_nodes, path, counts, nxt, dtype, ws, ws_bytes, None)
    assert call(batch=0) == 0
    for kw in (dict(logits=None), dict(tokens=None), dict(parents=None), dict(cu=None), dict(path=None), dict(counts=None), dict(nxt=None)):
        assert call(**kw) == NULL, kw
    for kw in (dict(batch=-1), dict(nodes=-1), dict(max_nodes=0), dict(max_nodes=65), dict(vocab=0), dict(stride=-1)):
        assert call(**kw) == SHAPE, kw
    for kw in (dict(logits=PTR + 1), dict(tokens=PTR + 4), dict(tokens=PTR + 2, i64=0), dict(nxt=PTR + 4), dict(path=PTR + 2)):
        assert call(**kw) == ALIGN, kw
    assert call(dtype=3) == DTYPE
    need = _lib().fn.en_accept_drafts_workspace_bytes
    assert need(5, 100, 1) > 0 and need(0, 100, 1) == 0 and need(4096, 130000, 1) == 0
    assert call(ws=None) == NULL and call(ws_bytes=need(5, 100, 1) - 1) == SHAPE and call(ws=PTR + 4) == ALIGN


def test_extension_refuses():
    fn = _lib().fn.en_kv_extend_paged

    def call(k=PTR, v=PTR, st=(128, 64) * 2, lens=PTR, cu=PTR, nodes=5, path=PTR, width=4, counts=PTR, **kw):
        return fn(k, v, None if st is None else (ctypes.c_int64 * 4)(*st), ctypes.byref(_pages(**kw)), lens, cu, nodes, path, width, counts, None, None)
    assert call(nodes=0) == 0 and call(width=0) == 0 and call(batch=0) == 0
    for kw in (dict(k=None), dict(v=None), dict(st=None), dict(lens=None), dict(cu=None), dict(path=None), dict(counts=None)):
        assert call(**kw) == NULL, kw
    for kw in (dict(nodes=-1), dict(width=65), dict(width=-1), dict(st=(-1, 64, 128, 64)), dict(head_num=0), dict(batch=1 << 17)):
        assert call(**kw) == SHAPE, kw
    assert call(dtype=4) == DTYPE and call(k=PTR + 1) == ALIGN and call(page_size=24) == UNSUPPORTED


def _w4(**kw):
    return _lib().W4(**{**dict(codes=PTR, scales=PTR, zeros=None, out_features=40, in_features=200, group=64, dtype=1), **kw})


def test_w4_refuses():
    lib = _lib()
    assert lib.fn.en_w4_codes_bytes(40, 200) == 3 * 2 * 1024 and lib.fn.en_w4_groups(40, 200, 64) == 3 * 2 * 2 * 16
    assert lib.fn.en_w4_codes_bytes(0, 8) == 0 and lib.fn.en_w4_groups(16, 128, 48) == 0

    def call(x=PTR, rows=4, stride=200, bias=None, act=0, y=PTR, ws=PTR, ws_bytes=1 << 40, **kw):
        return lib.fn.en_linear_w4(x, rows, stride, ctypes.byref(_w4(**kw)), bias, act, y, ws, ws_bytes, None)
    assert call(rows=0) == 0
    for kw in (dict(x=None), dict(y=None), dict(codes=None), dict(scales=None)):
        assert call(**kw) == NULL, kw
    assert lib.fn.en_linear_w4(PTR, 1, 200, None, None, 0, PTR, None, 0, None) == NULL
    for kw in (dict(rows=-1), dict(stride=192), dict(stride=-8), dict(out_features=0), dict(in_features=0), dict(in_features=204), dict(in_features=1 << 22), dict(rows=1 << 32)):
        assert call(**kw) == SHAPE, kw
    for kw in (dict(group=48), dict(act=4), dict(act=-1)):
        assert call(**kw) == UNSUPPORTED, kw
    for kw in (dict(x=PTR + 8), dict(stride=204), dict(codes=PTR + 8), dict(scales=PTR + 2), dict(zeros=PTR + 4), dict(y=PTR + 1), dict(bias=PTR + 1)):
        assert call(**kw) == ALIGN, kw
    for dtype in (0, 3):
        assert call(dtype=dtype) == DTYPE
    need = lib.fn.en_linear_w4_workspace_bytes
    assert need(1, 4096, 4096) == 0 and need(0, 4096, 4096) == 0 and need(40, 4096, 4096) > 0
    wide = dict(rows=40, stride=4096, out_features=4096, in_features=4096)
    assert call(ws=None, **wide) == NULL and call(ws_bytes=need(40, 4096, 4096) - 1, **wide) == SHAPE and call(ws=PTR + 8, **wide) == ALIGN
    pack = lib.fn.en_w4_pack
    assert pack(None, PTR, None, ctypes.byref(_w4()), None) == NULL and pack(PTR, PTR, PTR, ctypes.byref(_w4()), None) == NULL
    assert pack(PTR, PTR + 1, None, ctypes.byref(_w4()), None) == ALIGN and pack(PTR, PTR, None, ctypes.byref(_w4(group=16)), None) == UNSUPPORTED


def test_python_calls_refuse_host_tensors():
    from energonai_amd import kernel as K
    cpu = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.draft_tree(cpu, [4], 1)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.accept_drafts(torch.zeros(4, 9), cpu, None)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.w4_weight(torch.zeros(16, 64, dtype=torch.uint8), torch.zeros(16, 1, dtype=torch.float16))
    with pytest.raises(RuntimeError, match="W4Weight"):
        K.linear_w4(torch.zeros(1, 128, dtype=torch.float16), None)
    with pytest.raises(RuntimeError, match="multiple of 8"):
        K.w4_codes(torch.zeros(4, 12, dtype=torch.float16))


def test_codes_are_the_nearest():
    from energonai_amd import kernel as K
    g = torch.Generator().manual_seed(3)
    w = torch.randn(5, 200, generator=g).half()
    w[2, 64:128] = 0
    for zero_points in (False, True):
        codes, scales, zeros = K.w4_codes(w, 64, zero_points)
        assert codes.shape == (5, 100) and scales.shape == (5, 4) and (zeros is not None) == zero_points
        back, _ = ref.w4_values(codes, scales, zeros, 64)
        step = scales.double().repeat_interleave(64, 1)[:, :200]
        # half a step, or, where the range ends one code short or the scale and the zero point are themselves rounded, one and a half
        assert ((back - w.double()).abs() <= 1.51 * step + 1e-12).all()
        inside = (back - w.double()).abs() <= 0.51 * step + 1e-12
        assert inside.float().mean() > 0.95
        assert (back[2, 64:128] == 0).all() and (scales[2, 1] == 0)


def test_restatement_of_masks():
    m, d = ref.masks([-1, 0, 0, 1, 5, -1, 0], [5, 2])
    assert m == [1, 3, 5, 11, 16, 1, 3] and d == [0, 1, 1, 2, 0, 0, 1]


def test_sizes_past_64_bits_are_refused():
    """Products of sizes that pass 64 bits: no workspace for them, and strides that would come round to a small offset."""
    fn = _lib().fn
    assert fn.en_accept_drafts_workspace_bytes((1 << 31) - 1, (1 << 31) - 1, 0) == 0
    st = (ctypes.c_int64 * 6)(*(256, 64) * 3)
    far = (1 << 18, 1 << 14, 1 << 61, 1 << 18, 1 << 14, 64)
    c = _pages()
    for strides in (far, far[3:] + far[:3]):
        c.strides[:] = strides
        assert fn.en_decode_attn_tree(PTR, PTR, PTR, st, PTR, ctypes.byref(c), PTR, PTR, PTR, 5, 4, 4 * c.head_num, 0.1, PTR, 1 << 40, None) == SHAPE


def test_extension_with_a_largest_number_of_nodes_refuses():
    fn = _lib().fn.en_kv_extend_paged_nodes

    def call(nodes=5, most=4, path=PTR, width=4):
        return fn(PTR, PTR, (ctypes.c_int64 * 4)(*(128, 64) * 2), ctypes.byref(_pages()), PTR, PTR, nodes, most, path, width, PTR, None, None)
    assert call(nodes=0) == 0 and call(width=0) == 0 and call(path=None) == NULL
    for most in (-1, 65):
        assert call(most=most) == SHAPE
