"""Tails of the 8-bit cache whose page is none: zeros, as the full blocks of such a page."""
import pytest
import torch

from gpu_util import announce
from oracle import kv8 as ref
from test_gpu_kv8 import check_attention, deal_pages, new_cache, rows_of, to_gpu

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
I8, E4 = torch.int8, torch.float8_e4m3fn


def _K():
    import energonai_amd.kernel as K
    return K


# sequences, key heads, pages a sequence: a workgroup a unit; whole units to the waves; runs of tiles
@pytest.mark.parametrize("B,H,max_pages", [(6, 2, 4), (66, 8, 4), (6, 2, 80)])
@pytest.mark.parametrize("dtype,code,D,P", [(F16, I8, 64, 16), (BF16, E4, 80, 32), (F16, E4, 128, 64)])
@pytest.mark.parametrize("stale", ["NaN", "rows"])
def test_a_tail_without_a_page(B, H, max_pages, dtype, code, D, P, stale):
    """Attention and read-back, whatever the tail holds: NaN, or the rows of a sequence that had its place before."""
    K = _K()
    announce("kv8 tail without a page", B, H, max_pages, dtype, code, D, P, stale)
    g = torch.Generator().manual_seed(D)
    # only a tail; one behind a full block of its page; one whose page begins with it, behind a tile and a page of blocks; with a page
    some = [5, P + 15 if P == 16 else 31, P + 1, 2 * P + 3, P + 17 if P > 16 else 2 * P + 9, P]
    lens = [some[b % 6] for b in range(B)]
    cache = new_cache(B, H, D, P, sum(n // P + 1 for n in lens) + 1, max(max_pages, 1024 // P + 1 if max_pages > 4 else 0), dtype, code, g)
    deal_pages(cache, lens, P, g)
    ks, vs = rows_of(B, H, D, lens, dtype, g), rows_of(B, H, D, lens, dtype, g)
    for b in range(B):
        ref.put(cache, b, ks[b], vs[b])
    holes = []
    for b, n in enumerate(lens):
        if b % 6 != 4 and n % 16:
            pi = n // P
            cache[6][b, pi] = (-1, cache[0].shape[0], 1 << 30)[b % 3]
            holes.append((b, pi * P, n))
            if stale == "NaN":
                cache[4][b], cache[5][b] = float("nan"), float("nan")
    dev = to_gpu(cache)
    at = torch.tensor(lens, dtype=torch.int32).cuda()
    q = torch.randn(B, 2 * H, 1, D, generator=g).to(dtype)
    few = range(min(B, 6))
    got = K.decode_attn_kv8(q.cuda(), dev, at)
    check_attention(got[:6], q[:6], cache, lens[:6], ks[:6], vs[:6], code, D ** -0.5, "attention", holes)
    S, held = max(lens) + 3, ref.Cache(H, D, code)
    first = torch.tensor([max(0, n - 9) for n in lens], dtype=torch.int32)
    whole, window = K.kv8_pages_read(dev, at, S), K.kv8_pages_read(dev, at, 12, first=first.cuda())
    for b in few:
        for x, y, rows in ((whole[0], window[0], ks[b]), (whole[1], window[1], vs[b])):
            want = torch.zeros(H, S + 12, D, dtype=dtype)
            want[:, :lens[b]] = held.held(rows).float().to(dtype)
            for bb, lo, hi in holes:
                if bb == b:
                    want[:, lo:hi] = 0
            f = int(first[b])
            # (as numbers: e4m3 has a zero of either sign, and they are the same)
            assert torch.equal(x[b].cpu(), want[:, :S]) and torch.equal(y[b].cpu(), want[:, f:f + 12]), b


def test_the_place_of_another_sequence():
    """A place in the batch is taken over by a sequence for which no page was left: nothing of the one before is seen."""
    K = _K()
    announce("kv8 place taken over")
    g = torch.Generator().manual_seed(2)
    B, H, D, P = 2, 2, 64, 16
    dev = list(K.kv8_pages(4, B, H, P, D, 2, F16, "cuda"))
    dev[6][0], dev[6][1] = torch.tensor([0, 1]), torch.tensor([2, 3])
    x = torch.randn(20, 2 * H, D, generator=g).to(F16).cuda()
    K.kv8_pages_fill(x[:, :H], x[:, H:], dev, B, 10, torch.tensor([10, 10], dtype=torch.int32).cuda())
    dev[6][1] = -1
    over = torch.zeros(1, dtype=torch.int32, device="cuda")
    K.kv8_pages_fill(x[:, H:], x[:, :H], dev, B, 14, torch.tensor([6, 14], dtype=torch.int32).cuda(), overflow=over)
    assert int(over) == 14
    at = torch.tensor([6, 14], dtype=torch.int32).cuda()
    k, v = K.kv8_pages_read(dev, at, 16)
    assert torch.equal(k[0, :, :6], x[:6, H:].transpose(0, 1)) and bool((k[1] == 0).all()) and bool((v[1] == 0).all())
    q = torch.randn(B, H, 1, D, generator=g).to(F16).cuda()
    assert bool((K.decode_attn_kv8(q, dev, at)[1] == 0).all())
