"""What the C entry points of norm, rotation and the 8-bit cache refuse before anything reaches the device, and the plain restatement of
that cache that the GPU tests compare with."""
import ctypes

import pytest
import torch

from oracle import kv8 as ref

NULL, SHAPE, DTYPE, ALIGN = -1, -2, -3, -4
PTR = 1 << 20                                             # an address that nothing reads: every call here ends in a refusal or has nothing to do


def _lib():
    from energonai_amd import _lib as lib
    return lib


def _how(**kw):
    return _lib().NormRotary(**{**dict(cos=PTR, sin=PTR, table_rows=8, rotary_dim=64, interleaved=0, eps=1e-6), **kw})


def _cache(**kw):
    c = _lib().Kv8Cache(PTR, PTR, PTR, PTR, PTR, PTR, PTR)
    c.code_strides[:] = [4096, 2048, 4096, 2048]
    c.scale_strides[:] = [4, 2, 4, 2]
    for n, v in {**dict(num_pages=4, page_size=32, max_pages_per_seq=2, batch=3, head_num=2, size_per_head=64, code=0, dtype=1), **kw}.items():
        if n in ("code_strides", "scale_strides"):
            getattr(c, n)[:] = v
        else:
            setattr(c, n, v)
    return c


def test_structures_match_the_header():
    import os
    import re
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(root, "include", "energon_hip.h")).read(), flags=re.S)
    for struct, cls in (("en_norm_rotary", _lib().NormRotary), ("en_kv8_cache", _lib().Kv8Cache)):
        body = re.search(r"typedef struct %s \{(.*?)\}" % struct, text, flags=re.S).group(1)
        names = [re.sub(r"[\s*]|\[.*\]", "", n) for line in body.split(";") if line.strip() for n in re.sub(r"^\s*(const\s+)?\w+\s", "", line.strip()).split(",")]
        assert names == [f[0] for f in cls._fields_], struct


def test_norm_and_rotation_refuse():
    fn = _lib().fn.en_qk_norm_rotary
    strides = (ctypes.c_int64 * 8)(*[128, 64] * 4)

    def call(q=PTR, k=PTR, qo=PTR, ko=PTR, cu=PTR, pos=None, batch=1, tokens=4, hq=2, hk=2, D=64, st=strides, dtype=1, **how):
        return fn(q, k, qo, ko, cu, pos, batch, tokens, hq, hk, D, st, ctypes.byref(_how(**how)), dtype, None)
    assert call(tokens=0) == 0 and call(batch=0) == 0
    for kw in (dict(q=None), dict(k=None), dict(qo=None), dict(ko=None), dict(cu=None), dict(st=None), dict(cos=None), dict(sin=None)):
        assert call(**kw) == NULL, kw
    for kw in (dict(D=0), dict(D=257), dict(rotary_dim=63), dict(rotary_dim=66), dict(rotary_dim=-2), dict(table_rows=0), dict(table_rows=-1), dict(hq=0),
               dict(hk=-1), dict(tokens=-1), dict(batch=-1), dict(tokens=1 << 33)):
        assert call(**kw) == SHAPE, kw
    for dtype in (-1, 3):
        assert call(dtype=dtype) == DTYPE
    for kw in (dict(q=PTR + 1), dict(ko=PTR + 1), dict(q_weight=PTR + 1), dict(cos=PTR + 2)):
        assert call(**kw) == ALIGN, kw
    assert fn(PTR, PTR, PTR, PTR, PTR, None, 1, 4, 2, 2, 64, strides, None, 1, None) == NULL

    fn2 = _lib().fn.en_kv_append_paged_rotary
    six, three = (ctypes.c_int64 * 6)(*[128, 64] * 3), (ctypes.c_int64 * 3)(1024, 512, 32)

    def append(p=(PTR,) * 8, batch=1, hq=2, hk=2, pages=2, size=16, pool=4, D=64, st=six, ps=three, dtype=1, **how):
        return fn2(*p, batch, hq, hk, pages, size, pool, D, st, ps, ctypes.byref(_how(**how)), dtype, None, None)
    assert append(batch=0) == 0
    for i in range(8):
        assert append(p=tuple(None if j == i else PTR for j in range(8))) == NULL
    assert append(st=None) == append(ps=None) == NULL
    for kw in (dict(size=8), dict(size=24), dict(hq=0), dict(hk=0), dict(batch=-1), dict(pages=-1), dict(pool=-1), dict(D=300), dict(batch=1 << 30), dict(rotary_dim=128)):
        assert append(**kw) == SHAPE, kw


def test_cache_calls_refuse():
    fn = _lib().fn
    six, four = (ctypes.c_int64 * 6)(*[128, 64] * 3), (ctypes.c_int64 * 4)(*[128, 64] * 2)
    ws = fn.en_decode_attn_kv8_workspace_bytes(3, 4, 2, 1 << 16, 64)
    assert ws > 0 and fn.en_decode_attn_kv8_workspace_bytes(3, 5, 2, 1 << 16, 64) == fn.en_decode_attn_kv8_workspace_bytes(3, 4, 2, 64, 64) == 0
    how = _how()

    def calls(c):
        c = None if c is None else ctypes.byref(c)
        return [fn.en_kv8_fill(PTR, PTR, c, PTR, 4, 4, four, None, None), fn.en_kv8_append(PTR, PTR, PTR, PTR, c, PTR, 4, six, ctypes.byref(how), None, None),
                fn.en_kv8_read(c, PTR, None, 4, PTR, PTR, None), fn.en_decode_attn_kv8(PTR, PTR, c, PTR, 4, 1.0, PTR, ws, None)]
    assert calls(_cache(batch=0)) == [0] * 4
    assert calls(None) == [NULL] * 4
    assert calls(_cache(batch=0, page_table=None)) == [0] * 4 and calls(_cache(page_table=None)) == [NULL] * 4
    for n in ("k_pages", "v_pages", "k_scales", "v_scales", "k_tail", "v_tail", "page_table"):
        assert calls(_cache(**{n: None})) == [NULL] * 4, n
    for kw in (dict(num_pages=0), dict(page_size=8), dict(page_size=48), dict(max_pages_per_seq=-1), dict(batch=-1), dict(head_num=0), dict(size_per_head=40),
               dict(size_per_head=0), dict(size_per_head=144), dict(max_pages_per_seq=1 << 27), dict(code_strides=[1 << 32, 2048, 4096, 2048]),
               dict(scale_strides=[4, 2, -4, 2])):
        assert calls(_cache(**kw)) == [SHAPE] * 4, kw
    for kw in (dict(code=2), dict(dtype=0), dict(dtype=7)):
        assert calls(_cache(**kw)) == [DTYPE] * 4, kw
    for kw in (dict(k_pages=PTR + 8), dict(v_tail=PTR + 2), dict(k_scales=PTR + 2), dict(code_strides=[4096, 2056, 4096, 2048])):
        assert calls(_cache(**kw)) == [ALIGN] * 4, kw
    c = ctypes.byref(_cache())
    assert fn.en_kv8_fill(None, PTR, c, PTR, 4, 4, four, None, None) == NULL and fn.en_kv8_fill(PTR, PTR, c, PTR, 0, 4, four, None, None) == 0
    assert fn.en_kv8_fill(PTR, PTR, c, PTR, -1, 4, four, None, None) == SHAPE
    assert fn.en_kv8_append(None, PTR, PTR, PTR, c, PTR, 4, six, ctypes.byref(how), None, None) == NULL
    assert fn.en_kv8_append(PTR, PTR, PTR, PTR, c, PTR, 4, six, ctypes.byref(_how(rotary_dim=66)), None, None) == SHAPE
    assert fn.en_kv8_read(c, PTR, None, -1, PTR, PTR, None) == SHAPE and fn.en_kv8_read(c, PTR, None, 4, PTR + 8, PTR, None) == ALIGN
    for hq in (0, 1, 3, 5):
        assert fn.en_decode_attn_kv8(PTR, PTR, c, PTR, hq, 1.0, PTR, ws, None) == SHAPE
    long = ctypes.byref(_cache(max_pages_per_seq=1 << 11))
    assert fn.en_decode_attn_kv8(PTR, PTR, long, PTR, 4, 1.0, None, ws, None) == NULL
    assert fn.en_decode_attn_kv8(PTR, PTR, long, PTR, 4, 1.0, PTR, ws - 1, None) == SHAPE
    assert fn.en_decode_attn_kv8(PTR + 2, PTR, c, PTR, 4, 1.0, PTR, ws, None) == ALIGN


def test_python_calls_refuse_host_tensors():
    import energonai_amd.kernel as K
    x = torch.zeros(2, 2, 64, dtype=torch.float16)
    c = K.kv8_pages(2, 2, 2, 32, 64, 1, torch.float16, "cpu", torch.int8)
    assert [tuple(t.shape) for t in c] == [(2, 2, 32, 64), (2, 2, 2, 64, 16), (2, 2, 2), (2, 2, 2), (2, 2, 16, 64), (2, 2, 64, 16), (2, 1)]
    for call in (lambda: K.qk_norm_rotary(x, x, 1, [2]), lambda: K.kv_pages_append_rotary(x, x, x, x, x, [1, 1], c[6]),
                 lambda: K.kv8_pages_fill(x, x, c, 2, 1, [1, 1]), lambda: K.kv8_pages_append(x, x, x, c, [1, 1]),
                 lambda: K.kv8_pages_read(c, [1, 1], 1), lambda: K.decode_attn_kv8(x, c, [1, 1])):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()


def test_restated_cache():
    """Codes are the nearest, ties to even, by search over all of them; positions of a block that is not full are kept as they are."""
    g = torch.Generator().manual_seed(1)
    for code in (torch.int8, torch.float8_e4m3fn):
        every = torch.arange(-128, 128, dtype=torch.int8).view(code).float()
        every = every[every.abs() <= ref.LARGEST[code]].unique()
        x = torch.randn(16, 32, generator=g).half()
        x[0, :4] = torch.tensor([0.0, 1.0, -1.0, 0.5])
        c, s = ref.quantize(x, code)
        y = x.float() * (ref.LARGEST[code] / x.float().abs().max())
        near = (y[..., None] - every).abs().min(-1).values
        assert torch.equal((y - c.float()).abs(), near) and s == x.float().abs().max() / ref.LARGEST[code]
        held = ref.Cache(1, 32, code).held(torch.cat((x, x[:3]))[None])
        assert torch.equal(held[0, 16:], x[:3].double()) and torch.equal(held[0, :16], c.float().double() * s.double())


def test_results_over_rows_still_to_be_read():
    """Which results of the norm and rotation are refused, against the elements that views really share: what shares any is refused; of the
    layouts that projections have, what shares none is taken."""
    import random
    from energonai_amd.kernel.rotary import _apart, _not_over
    rng = random.Random(3)

    def elements(t):
        return {int(i) for i in (t.storage_offset() + sum(torch.arange(n).view([-1 if j == d else 1 for j in range(3)]) * s
                                                          for d, (n, s) in enumerate(zip(t.shape, t.stride())))).flatten()}
    base = torch.zeros(4000)
    shared = 0
    for _ in range(3000):
        D = rng.choice([1, 2, 4])
        views = []
        for _ in range(2):
            T, H = rng.randint(1, 4), rng.randint(1, 4)
            views.append(base.as_strided((T, H, D), (rng.choice([D, 2 * D, 3 * D, H * D, 4 * H * D, 50]), rng.choice([D, 2 * D, 3 * D, T * D, 50]), 1),
                                         rng.randint(0, 60)))
        if rng.random() < 0.5:                              # the same strides, as two parts of one projection have them
            views[1] = base.as_strided((views[0].shape[0], views[1].shape[1], D), views[0].stride(), views[1].storage_offset())
        a, b = views
        share = bool(elements(a) & elements(b))
        shared += share
        assert not (share and _apart(a, b)) and _apart(a, b) == _apart(b, a), (a.shape, a.stride(), b.shape, b.stride())
        if len(elements(a)) < a.numel():
            with pytest.raises(RuntimeError, match="overlap"):
                _not_over("t", [b], [a])
    assert 300 < shared < 2700
    x = torch.zeros(5, 3, 4, 8)
    three = [x[:, i] for i in range(3)]                     # [T, 3, H, D]
    of_heads = [x.view(5, 4, 3, 8)[:, :, i] for i in range(3)]
    for q, k, _ in (three, of_heads, [x[:1, i] for i in range(3)], [x.view(5, 4, 3, 8)[:1, :, i] for i in range(3)]):
        _not_over("t", [q, k], [q, k])
    q = x.view(5, 12, 8)
    for ins, outs in (([q[:, :8], q[:, 4:8]], [q[:, :8], q[:, 4:8]]), ([q, q], [q, torch.zeros(5, 12, 8)]), ([q[:4], q[1:]], [q[:4], torch.zeros(4, 12, 8)])):
        with pytest.raises(RuntimeError):
            _not_over("t", ins, outs)
