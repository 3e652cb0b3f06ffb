"""Sequences whose tiles many waves share: every tile counts, and counts once.

The keys are small, so that every position has about the same weight, and the values of 64 positions are large in one channel of their own: a
share that is lost, doubled or weighed wrongly moves that channel by many times the bound.  What is wanted comes from the codes as the
float32 definition gives them, not from the cache read back."""
import pytest
import torch

from gpu_util import announce
from oracle import kv8 as ref

F16, BF16 = torch.float16, torch.bfloat16
I8, E4 = torch.int8, torch.float8_e4m3fn
TILE = 64

CASES = [
    # dtype, code, Hq, H, D, lens
    (BF16, I8, 8, 1, 128, [70001]), (F16, E4, 8, 1, 128, [65536]),              # hundreds of waves a unit
    (F16, I8, 4, 2, 64, [30011, 16, 21000]), (BF16, E4, 17, 1, 80, [9000, 0, 12345, 64, 63]),      # two runs of queries a key head
]


def held(rows, code):
    """`oracle.kv8.Cache.held` of ``[H, n, D]`` rows, all blocks at once."""
    H, n, D = rows.shape
    full = n // 16 * 16
    out = rows.double().clone()
    if full:
        x = rows[:, :full].float().view(H, -1, 16, D)
        top = x.abs().amax((-1, -2), keepdim=True)
        m = torch.tensor(ref.LARGEST[code])
        some = top >= 2.0 ** -100
        y = torch.where(some, x * (m / top), 0.0)
        codes = (y.round() if code == I8 else y).to(code).float().double()
        out[:, :full] = (codes * torch.where(some, top / m, 0.0).double()).view(H, full, D)
    return out


def make(dtype, code, Hq, H, D, lens):
    g = torch.Generator().manual_seed(sum(lens))
    ks = [(0.02 * torch.randn(H, n, D, generator=g)).to(dtype) for n in lens]
    vs = []
    for n in lens:
        tile = torch.arange(n) // TILE
        v = 0.02 * torch.randn(H, n, D, generator=g)
        v[:, torch.arange(n), tile % D] += (8 + torch.randn(H, n, generator=g)) * (1 - 2.0 * (tile // D % 2))
        vs.append(v.to(dtype))
    return ks, vs, torch.randn(len(lens), Hq, 1, D, generator=g).to(dtype)


def wanted(q, k, v, scale):
    """(context, bound) of the queries ``[G, D]`` of a head over float64 keys and values: what `test_gpu_kv8.check_attention` allows."""
    D, half = q.shape[-1], torch.finfo(q.dtype).eps / 2
    want, size = ref.attention(q, k, v, scale)
    m = scale * (q.double().abs() @ k.abs().t()).max(-1, keepdim=True).values
    tol = half * (size + want.abs()) + (2 * (D / 8 + 4) * 2.0 ** -24 * m + 2.0 ** -18) * size + (2.0 ** -24 if q.dtype == F16 else 1e-38)
    if q.dtype == F16:
        tol = tol + 2.0 ** -25 * torch.softmax(q.double() @ k.t() * scale, -1).max(-1, keepdim=True).values * v.abs().sum(0)
    return want, tol


@pytest.mark.parametrize("dtype,code,Hq,H,D,lens", CASES)
def test_the_bound_sees_one_tile(dtype, code, Hq, H, D, lens):
    """Without any one tile, or with one twice, the result is out of bounds in some channel."""
    ks, vs, q = make(dtype, code, Hq, H, D, lens)
    assert torch.equal(held(ks[0][:, :200], code), ref.Cache(H, D, code).held(ks[0][:, :200]))
    b = max(range(len(lens)), key=lambda i: lens[i])
    k, v = held(ks[b], code)[0], held(vs[b], code)[0]
    qh = q[b, :1, 0]
    want, tol = wanted(qh, k, v, D ** -0.5)
    w = torch.exp(qh.double() @ k.t() * D ** -0.5)[0]
    tiles = -(-lens[b] // TILE)
    num = torch.zeros(tiles, D, dtype=torch.float64).index_add_(0, torch.arange(lens[b]) // TILE, w[:, None] * v)
    den = torch.zeros(tiles, dtype=torch.float64).index_add_(0, torch.arange(lens[b]) // TILE, w)
    for sign in (-1, 1):
        other = (num.sum(0) + sign * num[:-1]) / (den.sum() + sign * den[:-1])[:, None]      # the last one may be a few positions
        assert bool((((other - want).abs() - tol).amax(1) > 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,code,Hq,H,D,lens", CASES)
def test_every_tile_counts_once(dtype, code, Hq, H, D, lens):
    import energonai_amd.kernel as K
    announce("kv8 shares, tile by tile", dtype, code, Hq, H, D, lens)
    ks, vs, q = make(dtype, code, Hq, H, D, lens)
    B, P = len(lens), 64
    cache = list(K.kv8_pages(sum(n // P + 1 for n in lens), B, H, P, D, max(lens) // P + 2, dtype, "cuda", code))
    ids = torch.randperm(cache[0].shape[0], generator=torch.Generator().manual_seed(B)).tolist()
    table = torch.full(cache[6].shape, -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        for pi in range(-(-n // P)):
            table[b, pi] = ids.pop()
    cache[6] = table.cuda()
    at = torch.tensor(lens, dtype=torch.int32).cuda()
    pack = lambda xs: torch.cat([x.transpose(0, 1) for x in xs]).cuda()  # noqa: E731
    K.kv8_pages_fill(pack(ks), pack(vs), cache, B, max(lens), at)
    got = K.decode_attn_kv8(q.cuda(), cache, at).double().cpu()
    G = Hq // H
    for b, n in enumerate(lens):
        k, v = held(ks[b], code), held(vs[b], code)
        for h in range(H):
            rows = slice(h * G, (h + 1) * G)
            if n == 0:
                assert bool((got[b, rows] == 0).all())
                continue
            want, tol = wanted(q[b, rows, 0], k[h], v[h], D ** -0.5)
            off = ((got[b, rows, 0] - want).abs() - tol).max()
            assert off <= 0, (b, h, float(off))
