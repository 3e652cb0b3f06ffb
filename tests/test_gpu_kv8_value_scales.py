"""Decode attention over the 8-bit cache where the value scales of a query's blocks lie as far apart as they can: blocks whose values are all
zeros or next to nothing under the highest scores, and many small weights beside a large one."""
import math

import pytest
import torch

from gpu_util import announce
from oracle import kv8 as ref
from test_gpu_kv8 import check_attention, deal_pages, new_cache, to_gpu

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
I8, E4 = torch.int8, torch.float8_e4m3fn

# sequences, key heads, page size, pages a sequence: a workgroup a unit; whole units to the waves; runs of tiles
DEALS = {"team": (3, 2, 16, 12), "whole": (66, 8, 16, 12), "runs": (3, 2, 64, 32)}


def _K():
    import energonai_amd.kernel as K
    return K


def _fill(cache, ks, vs, lens):
    """The cache on the GPU, filled; a page that the table leaves out is filled as none."""
    dev = to_gpu(cache)
    pack = lambda xs: torch.cat([x.transpose(0, 1) for x in xs]).cuda()  # noqa: E731
    _K().kv8_pages_fill(pack(ks), pack(vs), dev, len(lens), max(lens), torch.tensor(lens, dtype=torch.int32).cuda())
    return dev


@pytest.mark.parametrize("deal", DEALS)
@pytest.mark.parametrize("dtype,code", [(F16, I8), (F16, E4), (BF16, I8), (BF16, E4)])
@pytest.mark.parametrize("kind", ["zeros", "no page", "next to nothing"])
def test_a_block_without_values_leads(deal, dtype, code, kind):
    """One block has the highest score by 90 to 400 and values that are zeros (of its own, or those of a page that is none), or 2^-90; the values
    of the others are around 1000 (bf16: once 2^100).  What the others add is exp of that less: nothing, and no infinity, no NaN."""
    K = _K()
    announce("kv8 lead without values", deal, dtype, code, kind)
    if kind == "next to nothing" and dtype == F16:
        kind = "smallest"                             # 2^-24
    g = torch.Generator().manual_seed(len(kind))
    B, H, P, max_pages = DEALS[deal]
    D, G, scale = 64, 2, 0.125
    u = torch.randint(0, 2, (D,), generator=g) * 2.0 - 1.0
    lens, ks, vs, leads = [], [], [], []
    for b in range(B):
        n, lead = (75, 163, 90)[b % 3], (0, 4, 2)[b % 3]      # its first, a later and its middle block
        ahead = (90.0, 130.0, 400.0)[b // 3 % 3] if b >= 3 else (130.0, 400.0, 90.0)[b]
        lens.append(n)
        leads.append(lead)
        rows = slice(16 * lead, 16 * lead + 16)
        k = 0.05 * torch.randn(H, n, D, generator=g)
        step = ahead / (8 * D * scale)                        # of a key along u: queries are 8 u
        if kind == "no page":                                 # its keys read as zeros: the others are that far below
            k = k - step * u
        else:
            k[:, rows] = k[:, rows] + step * u
        v = 1000.0 * (1 + 0.3 * torch.randn(H, n, D, generator=g))
        if dtype == BF16 and b % 2:
            v[:, -20:] *= 2.0 ** 90
        v[:, rows] = {"zeros": 0.0, "no page": 0.0, "next to nothing": 2.0 ** -90, "smallest": 2.0 ** -24}[kind] * torch.randint(1, 3, (H, 16, D), generator=g)
        ks.append(k.to(dtype))
        vs.append(v.to(dtype))
    cache = new_cache(B, H, D, P, B * max_pages + 1, max_pages, dtype, code, g)
    deal_pages(cache, lens, P, g)
    holes = []
    if kind == "no page":
        for b, lead in enumerate(leads):
            pi = 16 * lead // P
            cache[6][b, pi] = -1
            holes.append((b, pi * P, min((pi + 1) * P, lens[b] // 16 * 16)))
            # the whole page is without values, and its tail is not looked at here
            ks[b], vs[b] = ks[b][:, :lens[b] // 16 * 16], vs[b][:, :lens[b] // 16 * 16]
            lens[b] = lens[b] // 16 * 16
    dev = _fill(cache, ks, vs, lens)
    q = (8 * u + 0.01 * torch.randn(B, G * H, 1, D, generator=g)).to(dtype)
    got = K.decode_attn_kv8(q.cuda(), dev, torch.tensor(lens, dtype=torch.int32).cuda(), scale=scale)
    assert bool(torch.isfinite(got).all())
    for b in range(min(B, 9)):
        _check(got[[b]], q[[b]], lens[b], ks[b], vs[b], code, scale, [(0, lo, hi) for bb, lo, hi in holes if bb == b], (deal, kind, b))


def _check(got, q, n, k, v, code, scale, holes, what):
    """`check_attention` of one sequence, with room for weights of less than 2^-119 of the largest.  exp2 in fp32 has no normal numbers under
    2^-126, and the factor between a weight and its probability is a finite one, 2^128 at most, where up to 2^8 of it are left: what lies
    below 2^(8 - 128) may be off by all of itself."""
    held = ref.Cache(k.shape[0], k.shape[2], code)
    kd, vd = held.held(k), held.held(v)
    for _, lo, hi in holes:
        kd[:, lo:hi], vd[:, lo:hi] = 0, 0
    got = got.double().cpu().clone()
    G = q.shape[1] // k.shape[0]
    for h in range(k.shape[0]):
        rows = slice(h * G, (h + 1) * G)
        want, _ = ref.attention(q[0, rows, 0], kd[h], vd[h], scale)
        p = torch.softmax(q[0, rows, 0].double() @ kd[h].t() * scale, -1)
        room = torch.where(p < 2.0 ** -119 * p.amax(-1, keepdim=True), p, 0.0) @ vd[h].abs()
        off = got[0, rows, 0] - want
        got[0, rows, 0] = want + torch.sign(off) * (off.abs() - room).clamp_min(0)
    check_attention(got, q, None, [n], [k], [v], code, scale, what, holes)


@pytest.mark.parametrize("code", [I8, E4])
@pytest.mark.parametrize("n,capacity,B", [
    (1003, 1024, 1), (3000, 4096, 1), (60011, 65536, 1),      # the tiles of the sequence dealt to several waves
    (4096, 4096, 1100), (240, 256, 600),                      # one wave has all of them: many sequences, on the same pages
])
def test_many_small_weights_beside_a_large_one(code, n, capacity, B):
    """fp16: one position has a weight 2^26 times that of each of the others, whose values make up the result all the same where the one's
    is zero.  A weight is rounded to fp16 for its product with the values; that leaves 2^-32 of the largest: numbers there go down to
    2^-24, half of that is lost, and the largest stands at 2^7 or above."""
    K = _K()
    announce("kv8 small weights", code, n, capacity, B)
    g = torch.Generator().manual_seed(n)
    D, H, P, scale = 64, 1, 64, 0.125
    u = torch.randint(0, 2, (D,), generator=g) * 2.0 - 1.0
    k = torch.zeros(H, n, D)
    k[:, 37] = 26 * math.log(2) / (8 * D * scale) * u
    v = 50.0 * (1 + 0.2 * torch.randn(H, n, D, generator=g)) * (torch.arange(D) % 2 * 2 - 1)
    v[:, 37, :32] = 0.0
    ks, vs = [k.to(F16)], [v.to(F16)]
    cache = new_cache(1, H, D, P, n // P + 2, capacity // P, F16, code, g)
    deal_pages(cache, [n], P, g)
    dev = _fill(cache, ks, vs, [n])
    dev[4:] = [t.expand(B, *t.shape[1:]).contiguous() for t in dev[4:]]
    q = (8 * u).expand(B, 2, 1, D).to(F16)
    got = K.decode_attn_kv8(q.cuda(), dev, torch.full((B,), n, dtype=torch.int32).cuda(), scale=scale).double().cpu()[:, :, 0]
    q = q[0, :, 0]
    held = ref.Cache(H, D, code)
    kd, vd = held.held(ks[0])[0], held.held(vs[0])[0]
    want, size = ref.attention(q, kd, vd, scale)
    m = scale * (q.double().abs() @ kd.abs().t()).max(-1, keepdim=True).values
    # check_attention's bound with 2^-32 where that has 2^-25
    tol = 2.0 ** -11 * (size + want.abs()) + 2.0 ** -24 + (2 * (D / 8 + 4) * 2.0 ** -24 * m + 2.0 ** -18) * size \
        + 2.0 ** -32 * torch.softmax(q.double() @ kd.t() * scale, -1).max() * vd.abs().sum(0)
    off = ((got - want).abs() - tol).amax((1, 2))
    assert off.max() <= 0, (int(off.argmax()), float(off.max()))
    assert bool((want[:, :32].abs() > 8 * tol[:, :32]).all())         # what the others come to is far more than the bound
