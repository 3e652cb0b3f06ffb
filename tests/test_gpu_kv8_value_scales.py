"""Decode attention over the 8-bit cache where the value scales of a query's blocks lie as far apart as they can: blocks whose values are all
zeros or next to nothing under the highest scores."""
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
