"""Norm and rotation, fills and reads of the 8-bit cache that are large enough to go past the caches: the bits of the same rows in small calls.

The sizes lie just past those from which stores (96 MiB) and loads (384 MiB) are non-temporal."""
import pytest
import torch

from gpu_util import announce
from test_gpu_kv8 import same_bits

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
I8, E4 = torch.int8, torch.float8_e4m3fn


def _K():
    import energonai_amd.kernel as K
    return K


@pytest.mark.parametrize("dtype,Hq,Hk,D,R,il,mb", [
    (BF16, 32, 8, 128, 128, False, 100), (BF16, 32, 8, 128, 128, False, 390), (F16, 24, 24, 64, 64, True, 390), (F16, 12, 5, 80, 20, False, 390),
    (F32, 16, 3, 96, 48, True, 100), (F32, 16, 3, 96, 96, False, 390), (F16, 10, 2, 50, 6, True, 100), (F16, 10, 2, 50, 6, False, 390),
])
def test_qk_norm_rotary(dtype, Hq, Hk, D, R, il, mb):
    K = _K()
    announce("qk_norm_rotary, large", dtype, Hq, Hk, D, R, il, mb)
    T = (mb << 20) // ((Hq + Hk) * D * dtype.itemsize) + 77
    g = torch.Generator(device="cuda").manual_seed(mb + D)
    x = torch.randn(T + 3, (Hq + Hk) * D, generator=g, device="cuda").to(dtype)
    q, k = (t.unflatten(1, (-1, D)) for t in x.split((Hq * D, Hk * D), 1))
    gains = [(1 + 0.1 * torch.randn(D, generator=g, device="cuda")).to(dtype) for _ in range(2)]
    lens = [T // 3, 0, 1, T - T // 3 - 1 - 500, 500]
    rot = K.rotary_table(max(lens), R)
    kw = dict(q_weight=gains[0], k_weight=gains[1], interleaved=il)
    out = tuple(torch.full(t.shape, 7.0, dtype=dtype, device="cuda") for t in (q, k))
    K.qk_norm_rotary(q, k, len(lens), torch.tensor(lens, dtype=torch.int32).cuda(), rot, out=out, **kw)
    assert all(bool((t[T:] == 7.0).all()) for t in out)
    pos = torch.cat([torch.arange(n, dtype=torch.int32) for n in lens]).cuda()
    step = 200                                        # under 16384 rows a call
    for t in range(0, T, step):
        rows = slice(t, min(t + step, T))
        want = K.qk_norm_rotary(q[rows], k[rows], 0, None, rot, positions=pos[rows], **kw)
        assert torch.equal(out[0][rows], want[0]) and torch.equal(out[1][rows], want[1]), t


@pytest.mark.parametrize("dtype,code,H,D,P", [(BF16, E4, 64, 128, 64), (F16, I8, 40, 64, 128), (F16, E4, 24, 80, 32)])
def test_kv8_fill_and_read(dtype, code, H, D, P):
    K = _K()
    announce("kv8 fill and read, large", dtype, code, H, D, P)
    T = (390 << 20) // (4 * H * D)
    lens = [T // 4 + 5, 1, T // 2, 0, 37, T - T // 4 - 5 - 1 - T // 2 - 37]
    B, S = len(lens), max(lens)
    pages = [-(-n // P) for n in lens]
    g = torch.Generator(device="cuda").manual_seed(D)
    kv = torch.randn(T, 2 * H, D, generator=g, device="cuda").to(dtype)
    large = list(K.kv8_pages(sum(pages) + 1, B, H, P, D, max(pages), dtype, "cuda", code))
    ids = torch.randperm(sum(pages), generator=torch.Generator().manual_seed(P)).tolist()
    table = torch.full(large[6].shape, -1, dtype=torch.int32)
    for b, n in enumerate(pages):
        for pi in range(n):
            table[b, pi] = ids.pop()
    large[6] = table.cuda()
    small = list(K.kv8_pages(sum(pages) + 1, B, H, P, D, max(pages), dtype, "cuda", code))
    small[6] = large[6]
    at = torch.tensor(lens, dtype=torch.int32).cuda()
    K.kv8_pages_fill(kv[:, :H], kv[:, H:], large, B, S, at)
    # the same in pieces of whole pages, a sequence at a time: its row of the table from there on, and its tail
    start = 0
    chunk = max(P, 1024)
    for b, n in enumerate(lens):
        for p in range(0, n, chunk):
            rows = kv[start + p:start + min(p + chunk, n)]
            part = small[:4] + [small[4][b:b + 1], small[5][b:b + 1], small[6][b:b + 1, p // P:].contiguous()]
            K.kv8_pages_fill(rows[:, :H], rows[:, H:], part, 1, rows.shape[0], torch.tensor([rows.shape[0]], dtype=torch.int32).cuda())
        start += n
    for name, a, b in zip(K.KV8Pages._fields, large, small):
        assert same_bits(a, b), name
    k, v = K.kv8_pages_read(large, at, S)
    for s in range(0, S, 500):
        n = min(500, S - s)
        k2, v2 = K.kv8_pages_read(large, at, n, first=torch.full((B,), s, dtype=torch.int32).cuda())
        assert torch.equal(k[:, :, s:s + n], k2) and torch.equal(v[:, :, s:s + n], v2), s
