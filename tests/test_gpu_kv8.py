"""The K/V cache in 8 bits: what is written, bit for bit; what is read; and the decode attention over it, against float64."""
import pytest
import torch

from gpu_util import announce
from oracle import kv8 as ref

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
I8, E4 = torch.int8, torch.float8_e4m3fn


def _K():
    import energonai_amd.kernel as K
    return K


def new_cache(B, H, D, P, N, max_pages, dtype, code, g, garbage=True):
    """A cache on the CPU whose bytes are anything: every code (e4m3: NaN among them), NaN scales, NaN tails."""
    blocks = P // 16
    codes = lambda *s: torch.randint(-128, 128, s, generator=g, dtype=torch.int8).view(code) if garbage else torch.zeros(s, dtype=torch.int8).view(code)  # noqa: E731
    fill = float("nan") if garbage else 0.0
    return [codes(N, H, P, D), codes(N, H, blocks, D, 16), torch.full((N, H, blocks), fill), torch.full((N, H, blocks), fill),
            torch.full((B, H, 16, D), fill, dtype=dtype), torch.full((B, H, D, 16), fill, dtype=dtype),
            torch.full((B, max_pages), -1, dtype=torch.int32)]


def deal_pages(cache, lens, P, g, room=0):
    """Distinct pages in any order for positions 0 .. len + room - 1."""
    ids = torch.randperm(cache[0].shape[0], generator=g).tolist()
    for b, n in enumerate(lens):
        for pi in range(-(-(n + room) // P)):
            cache[6][b, pi] = ids.pop()


def to_gpu(cache):
    return [t.cuda() for t in cache]


def same_bits(a, b):
    a, b = a.cpu(), b.cpu()
    if a.dtype.itemsize == 1:
        return torch.equal(a.view(torch.int8), b.view(torch.int8))
    return torch.equal(a.view(torch.int16) if a.dtype.itemsize == 2 else a.view(torch.int32), b.view(torch.int16) if b.dtype.itemsize == 2 else b.view(torch.int32))


def rows_of(B, H, D, lens, dtype, g, size=1.0):
    """Per sequence [H, n, D] rows whose channels differ in size."""
    channel = torch.exp(0.7 * torch.randn(D, generator=g)) * size
    return [(torch.randn(H, n, D, generator=g) * channel).to(dtype) for n in lens]


FILL = [
    # dtype, code, H, D, P, lens
    (F16, I8, 1, 64, 16, [1]), (F16, I8, 12, 64, 64, [700, 9, 64, 16, 15, 0, 33]), (BF16, E4, 8, 128, 128, [300, 17, 128]),
    (BF16, I8, 3, 80, 32, [50, 32, 47]), (F16, E4, 2, 96, 16, [31, 48]), (BF16, E4, 5, 112, 64, [65, 1]), (F16, I8, 2, 16, 16, [40]),
    (F16, E4, 3, 32, 32, [40, 16]), (BF16, I8, 1, 48, 16, [33]),
]


@pytest.mark.parametrize("dtype,code,H,D,P,lens", FILL)
def test_fill_append_read(dtype, code, H, D, P, lens):
    """A prompt's rows, bit for bit as the float32 definition holds them; nothing else written; the same cache from a shorter prompt and
    appends; and the positions read back."""
    K = _K()
    announce("kv8 fill/append/read", dtype, code, H, D, P, lens)
    g = torch.Generator().manual_seed(D + H + len(lens))
    B, S = len(lens), max(lens)
    max_pages = S // P + 2
    cache = new_cache(B, H, D, P, sum(n // P + 2 for n in lens) + 3, max_pages, dtype, code, g)
    deal_pages(cache, lens, P, g, room=1)
    ks, vs = rows_of(B, H, D, lens, dtype, g), rows_of(B, H, D, lens, dtype, g, 3.0)
    if lens[0] >= 16:
        ks[0][0, 3] *= 40                               # a row that is much larger than its block
        vs[0][0, :16] = 0                               # a block of zeros
    dev = to_gpu(cache)
    for b in range(B):
        ref.put(cache, b, ks[b], vs[b])
    pack = lambda xs: torch.cat([x.transpose(0, 1) for x in xs])  # noqa: E731
    kv = torch.cat((pack(ks), pack(vs)), 1).cuda()
    lens_t = torch.tensor(lens, dtype=torch.int32).cuda()
    over = torch.zeros(1, dtype=torch.int32, device="cuda")
    K.kv8_pages_fill(kv[:, :H], kv[:, H:], dev, B, S, lens_t, overflow=over)
    for name, a, b in zip(K.KV8Pages._fields, dev, cache):
        assert same_bits(a, b), name
    assert int(over) == 0
    # a prompt of the first third and then one position a step
    part = [n // 3 for n in lens]
    other = to_gpu(new_cache(B, H, D, P, cache[0].shape[0], max_pages, dtype, code, g))
    other[6] = dev[6]
    kv3 = torch.cat((pack([k[:, :n] for k, n in zip(ks, part)]), pack([v[:, :n] for v, n in zip(vs, part)])), 1).cuda()
    now = torch.tensor(part, dtype=torch.int32).cuda()
    K.kv8_pages_fill(kv3[:, :H], kv3[:, H:], other, B, max(part), now.clone())
    bound = dev[6].clone()
    for step in range(max(n - m for n, m in zip(lens, part)) if S <= 130 else 33):
        todo = [m + step < n for m, n in zip(part, lens)]
        new = torch.stack([torch.stack([x[b][:, part[b] + step] if todo[b] else torch.zeros(H, D, dtype=dtype) for b in range(B)]) for x in (ks, vs)]).cuda()
        other[6] = torch.where(torch.tensor(todo).cuda()[:, None], bound, -1)             # those that are done have no page
        K.kv8_pages_append(None, new[0], new[1], other, now, overflow=over.zero_())
        assert int(over) == B - sum(todo)
        now += torch.tensor(todo, dtype=torch.int32).cuda()
    other[6] = bound
    reached = now.tolist()
    held = ref.Cache(H, D, code)
    for c, n in ((dev, lens), (other, reached)):
        n_t = torch.tensor(n, dtype=torch.int32).cuda()
        k, v = K.kv8_pages_read(c, n_t, S + 5)
        first = torch.tensor([max(0, m - 21) for m in n], dtype=torch.int32)
        k2, v2 = K.kv8_pages_read(c, n_t, 19, first=first.cuda())
        for b, m in enumerate(n):
            for got, got2, rows in ((k, k2, ks[b]), (v, v2, vs[b])):
                want = torch.zeros(H, S + 40, D, dtype=dtype)
                want[:, :m] = held.held(rows[:, :m]).float().to(dtype)
                assert same_bits(got[b], want[:, :S + 5].contiguous()), b
                f = int(first[b])
                assert same_bits(got2[b], want[:, f:f + 19].contiguous()), b
    if reached == list(lens):
        blk = [(b, j) for b, n in enumerate(lens) for j in range(n // 16)]
        for b, j in blk:
            pid, r = int(bound[b, j * 16 // P]), j * 16 % P
            assert same_bits(other[0][pid, :, r:r + 16].contiguous(), dev[0][pid, :, r:r + 16].contiguous())
            assert same_bits(other[1][pid, :, r // 16].contiguous(), dev[1][pid, :, r // 16].contiguous())
            assert torch.equal(other[2][pid, :, r // 16], dev[2][pid, :, r // 16]) and torch.equal(other[3][pid, :, r // 16], dev[3][pid, :, r // 16])


def test_values_a_block_cannot_hold():
    """Infinities and NaN make their block's scale NaN, values under 2^-100 are zeros, and neither touches a neighbour."""
    K = _K()
    announce("kv8 odd values")
    g = torch.Generator().manual_seed(0)
    H, D, P = 3, 64, 64
    for code in (I8, E4):
        k = torch.randn(H, 64, D, generator=g).to(BF16)
        k[0, 3, 5], k[1, 20, 0], k[2, 40] = float("inf"), float("nan"), float("-inf")
        k[0, 48:] *= 2.0 ** -120
        k[1, 48:] *= 1e30
        cache = new_cache(1, H, D, P, 2, 1, BF16, code, g)
        cache[6][0, 0] = 1
        dev = to_gpu(cache)
        ref.put(cache, 0, k, k)
        rows = k.transpose(0, 1).contiguous().cuda()
        K.kv8_pages_fill(rows, rows, dev, 1, 64, [64])
        for name, a, b in zip(K.KV8Pages._fields, dev, cache):
            if a.dtype == torch.float32:
                assert torch.equal(torch.isnan(a).cpu(), torch.isnan(b)) and torch.equal(torch.nan_to_num(a).cpu(), torch.nan_to_num(b)), name
            else:
                assert same_bits(a, b), name


def test_fill_without_pages_and_strided():
    """Blocks without a page are left out and counted; pools may be two halves of one, rows any views."""
    K = _K()
    announce("kv8 fill without pages")
    g = torch.Generator().manual_seed(4)
    B, H, D, P = 3, 2, 64, 32
    lens = [70, 40, 5]
    cache = new_cache(B, H, D, P, 9, 3, F16, I8, g)
    deal_pages(cache, lens, P, g)
    cache[6][0, 1] = -1
    cache[6][1, 0] = 9
    cache[6][2, 0] = 1 << 30
    both = torch.stack((cache[0], cache[1].view(9, H, P, D)), 1).cuda()
    scales = torch.stack((cache[2], cache[3]), 1).cuda()
    dev = to_gpu(cache)
    dev[0], dev[1], dev[2], dev[3] = both[:, 0], both[:, 1].view(9, H, P // 16, D, 16), scales[:, 0], scales[:, 1]
    ks, vs = rows_of(B, H, D, lens, F16, g), rows_of(B, H, D, lens, F16, g)
    for b in range(2):
        ref.put(cache, b, ks[b], vs[b])
    wide = torch.zeros(sum(lens), 2 * H, D + 3, dtype=F16)
    wide[:, 0::2, :D] = torch.cat([x.transpose(0, 1) for x in ks])
    wide[:, 1::2, 3:] = torch.cat([x.transpose(0, 1) for x in vs])
    wide = wide.cuda()
    over = torch.zeros(1, dtype=torch.int32, device="cuda")
    K.kv8_pages_fill(wide[:, 0::2, :D], wide[:, 1::2, 3:], dev, B, 100, torch.tensor(lens, dtype=torch.int32).cuda(), overflow=over)
    assert int(over) == 32 + 32 + 5
    for name, a, b in zip(K.KV8Pages._fields, dev, cache):
        assert same_bits(a.contiguous(), b), name
    # a bucket shorter than a sequence takes what fits into it
    dev2 = to_gpu(cache)
    short = new_cache(B, H, D, P, 9, 3, F16, I8, g)
    short[6] = cache[6]
    dev2 = to_gpu(short)
    ref.put(short, 0, ks[0][:, :20], vs[0][:, :20])
    ref.put(short, 1, ks[1][:, :20], vs[1][:, :20])
    short[4][1], short[5][1] = float("nan"), float("nan")          # its first page is none
    K.kv8_pages_fill(wide[:, 0::2, :D], wide[:, 1::2, 3:], dev2, B, 20, torch.tensor(lens, dtype=torch.int32).cuda())
    for name, a, b in zip(K.KV8Pages._fields, dev2, short):
        assert same_bits(a, b), name


@pytest.mark.parametrize("dtype,code,Hq,H,D,R,il,norm", [
    (F16, I8, 12, 12, 64, 64, False, False), (BF16, E4, 16, 2, 128, 128, False, True), (BF16, I8, 3, 3, 80, 20, True, True),
    (F16, E4, 5, 1, 112, 14, False, True), (F16, I8, 2, 2, 16, 16, True, False),
])
def test_append_turns(dtype, code, Hq, H, D, R, il, norm):
    """Queries and keys normed and turned, to the nearest number of their type; keys in the tails and, where they complete a block, in the pages."""
    K = _K()
    announce("kv8 append turns", dtype, code, Hq, H, D, R, il, norm)
    g = torch.Generator().manual_seed(D)
    B, P = 20, 32
    lens = [0, 15, 31, 14, 16, 63] + torch.randint(0, 95, (B - 6,), generator=g).tolist()
    cache = new_cache(B, H, D, P, 3 * B + 1, 3, dtype, code, g)
    deal_pages(cache, lens, P, g, room=1)
    ks, vs = rows_of(B, H, D, lens, dtype, g), rows_of(B, H, D, lens, dtype, g)
    for b in range(B):
        ref.put(cache, b, ks[b], vs[b])
    dev = to_gpu(cache)
    x = torch.randn(B, (Hq + 2 * H) * D + 1, generator=g).to(dtype)[:, 1:].unflatten(1, (Hq + 2 * H, D)).cuda()
    q, k, v = x[:, :Hq], x[:, Hq:Hq + H], x[:, Hq + H:]
    gains = [(1 + 0.1 * torch.randn(D, generator=g)).to(dtype).cuda() if norm else None for _ in range(2)]
    rot = K.rotary_table(100, R)
    at = torch.tensor(lens, dtype=torch.int32).cuda()
    kw = dict(q_weight=gains[0], k_weight=gains[1], interleaved=il)
    got = K.kv8_pages_append(q, k, v, dev, at, rot, **kw)
    turned = torch.stack([dev[4][b, :, lens[b] % 16] for b in range(B)])
    for y, r, w, fp in ((got, q, gains[0], 32 * 2.0 ** -24), (turned, k, gains[1], 2.0 ** -40)):
        want, size = ref.norm_rotary(r.cpu(), at.cpu().long(), tuple(t.cpu() for t in rot), None if w is None else w.cpu(), 1e-6, il)
        # half a step of the type, and of its smallest numbers; keys are computed in 64 bits, queries in 32 (as in test_gpu_rotary.assert_rows)
        assert bool(((y.double().cpu() - want).abs() <= torch.finfo(dtype).eps / 2 * want.abs() + fp * size + (2.0 ** -25 if dtype == F16 else 0.0)).all())
    for b in range(B):
        n = lens[b]
        ref.put(cache, b, torch.cat((ks[b], turned[b].cpu()[:, None]), 1), torch.cat((vs[b], v[b].cpu()[:, None]), 1))
        if n % 16 == 15:                               # the tail keeps its last row
            cache[4][b, :, 15], cache[5][b, :, :, 15] = turned[b].cpu(), v[b].cpu()
    for name, a, b in zip(K.KV8Pages._fields, dev, cache):
        assert same_bits(a, b), name


def check_attention(got, q, cache, lens, ks, vs, code, scale, what, zero_pages=()):
    """The bounds of what the kernel rounds, each half a step:
    - the result, of its type: half |want|;
    - a probability (times its value scale), of the same type: half sum p |v|; fp16 has no steps under 2^-24, so one of its size there is off
      by 2^-25 of the largest: 2^-25 max p sum |v|;
    - a score in fp32: a sum of D exact products, 32 an instruction and at most four roundings each, D / 8, its factors and the
      difference to the maximum, 4: (D / 8 + 4) 2^-24 of m = scale max sum |q k|, and exp of it that much off, relative, above and below the line;
    - exp2 (a step), sums of up to 2^6 numbers a lane and the rest: 2^-18 of sum p |v|."""
    got = got.double().cpu()
    half = torch.finfo(q.dtype).eps / 2
    B, Hq, _, D = q.shape
    H = ks[0].shape[0]
    held = ref.Cache(H, D, code)
    for b, n in enumerate(lens):
        k, v = held.held(ks[b]), held.held(vs[b])
        for lo, hi in [(lo, hi) for bb, lo, hi in zero_pages if bb == b]:
            k[:, lo:hi], v[:, lo:hi] = 0, 0
        for h in range(H):
            rows = slice(h * (Hq // H), (h + 1) * (Hq // H))
            want, size = ref.attention(q[b, rows, 0], k[h], v[h], scale)
            tol = half * (size + want.abs()) + (2.0 ** -24 if q.dtype == F16 else 1e-38)
            if n:
                m = abs(scale) * (q[b, rows, 0].double().abs() @ k[h].abs().t()).max(-1, keepdim=True).values
                tol += (2 * (D / 8 + 4) * 2.0 ** -24 * m + 2.0 ** -18) * size
                if q.dtype == F16:
                    most = torch.softmax(q[b, rows, 0].double() @ k[h].t() * scale, -1).max(-1, keepdim=True).values
                    tol += 2.0 ** -25 * most * v[h].abs().sum(0)
            off = ((got[b, rows, 0] - want).abs() - tol).max()
            assert off <= 0, (what, b, n, h, float(off))


ATTEND = [
    # dtype, code, Hq, H, D, P, lens, size of q
    (F16, I8, 12, 12, 64, 16, [100], 2.0),
    (BF16, E4, 32, 8, 128, 64, [1, 15, 16, 17, 0, 63, 64, 65, 128, 200], 2.0),
    (F16, E4, 8, 8, 128, 64, [1000, 3, 517], 2.0),
    (BF16, I8, 20, 4, 80, 32, [400, 33, 0, 95], 1.0),
    (F16, I8, 7, 1, 96, 16, [300, 31], 4.0),
    (BF16, E4, 16, 1, 112, 128, [260, 128], 1.0),
    (F16, E4, 71, 1, 64, 64, [150, 5], 2.0),               # 71 queries a key head: five runs of 16
    (BF16, I8, 48, 2, 128, 64, [333], 2.0),                # 24
    (F16, I8, 3, 3, 16, 16, [70, 16], 1.0),
    (BF16, E4, 4, 2, 32, 32, [77], 1.0),
    (F16, E4, 2, 1, 48, 16, [90, 48], 1.0),
    (F16, I8, 4, 2, 128, 256, [5000, 77], 2.0),
]


@pytest.mark.parametrize("dtype,code,Hq,H,D,P,lens,size", ATTEND)
def test_attention(dtype, code, Hq, H, D, P, lens, size):
    K = _K()
    announce("decode_attn_kv8", dtype, code, Hq, H, D, P, lens)
    g = torch.Generator().manual_seed(D + Hq)
    B = len(lens)
    cache = new_cache(B, H, D, P, sum(n // P + 1 for n in lens) + 2, max(lens) // P + 2, dtype, code, g)
    deal_pages(cache, lens, P, g)
    ks, vs = rows_of(B, H, D, lens, dtype, g), rows_of(B, H, D, lens, dtype, g, 2.0)
    for b in range(B):
        ref.put(cache, b, ks[b], vs[b])
    q = (size * torch.randn(B, Hq, 1, D, generator=g)).to(dtype)
    dev = to_gpu(cache)
    at = torch.tensor(lens, dtype=torch.int32).cuda()
    scale = 0.6 * D ** -0.5
    out = torch.full((B, Hq, 1, D), 7.0, dtype=dtype, device="cuda")
    got = K.decode_attn_kv8(q.cuda(), dev, at, scale=scale, out=out)
    assert got is out
    check_attention(got, q, cache, lens, ks, vs, code, scale, "attention")
    ws = torch.full((K.decode_attn_kv8_workspace_bytes(B, Hq, H, cache[6].shape[1] * P, D),), 0xff, dtype=torch.uint8, device="cuda")
    assert torch.equal(K.decode_attn_kv8(q.cuda()[:, :, 0], K.KV8Pages(*dev), at, scale=scale, workspace=ws), got)      # whatever the workspace held
    for s in (-0.3, 0.0):
        check_attention(K.decode_attn_kv8(q.cuda(), dev, at, scale=s), q, cache, lens, ks, vs, code, s, s)


def test_attention_without_pages():
    """Positions on pages outside the pool read as zero keys and values; those behind the lengths as nothing."""
    K = _K()
    announce("decode_attn_kv8 without pages")
    g = torch.Generator().manual_seed(8)
    B, Hq, H, D, P = 3, 4, 2, 64, 16
    lens = [200, 100, 37]
    for dtype, code in ((F16, E4), (BF16, I8)):
        cache = new_cache(B, H, D, P, 40, 14, dtype, code, g)
        deal_pages(cache, lens, P, g)
        ks, vs = rows_of(B, H, D, lens, dtype, g), rows_of(B, H, D, lens, dtype, g)
        for b in range(B):
            ref.put(cache, b, ks[b], vs[b])
        cache[6][0, 3], cache[6][1, 0], cache[6][2, 1] = -1, 40, 1 << 30
        q = torch.randn(B, Hq, 1, D, generator=g).to(dtype)
        got = K.decode_attn_kv8(q.cuda(), to_gpu(cache), torch.tensor(lens, dtype=torch.int32).cuda())
        check_attention(got, q, cache, lens, ks, vs, code, D ** -0.5, "no pages", [(0, 48, 64), (1, 0, 16), (2, 16, 32)])
        # lengths past what the table can name end there; negative ones are none
        got = K.decode_attn_kv8(q.cuda(), to_gpu(cache), torch.tensor([1 << 30, -5, 0], dtype=torch.int32).cuda())
        assert bool((got[1:] == 0).all())


@pytest.mark.parametrize("D", [48, 64, 80, 112, 128])
def test_an_infinite_key_in_the_tail(D):
    """A key whose score is minus infinity is a masked one, as long as its block is in 16 bits; of any head size."""
    K = _K()
    announce("kv8 attention, infinite key", D)
    g = torch.Generator().manual_seed(D)
    H, n = 2, 21
    cache = new_cache(1, H, D, 16, 3, 2, F16, I8, g, garbage=False)
    deal_pages(cache, [n], 16, g)
    k, v = (torch.randn(n, H, D, generator=g).to(F16) for _ in range(2))
    q = torch.randn(1, H, 1, D, generator=g).to(F16)
    q[0, :, 0, 0] = -1.0
    k[18, :, 0] = float("inf")
    gpu = to_gpu(cache)
    from energonai_amd.seqinfo import build_seq_info
    info = build_seq_info(torch.tensor([n], dtype=torch.int32, device="cuda"), 1)
    K.kv8_pages_fill(k.cuda(), v.cuda(), gpu, 1, n, info)
    got = K.decode_attn_kv8(q.cuda(), gpu, info)
    kd, vd = (t.cpu().double() for t in K.kv8_pages_read(gpu, info, n))
    kd[0, :, 18] = 0
    s = (q[0, :, 0].double()[:, None] * kd[0]).sum(-1) * D ** -0.5
    s[:, 18] = float("-inf")
    want = (torch.softmax(s, -1)[..., None] * vd[0]).sum(1)
    # half steps of 2^-11: of the keys as they are read here (a score is off by e, a probability by 2 e), of the values as they are read, of
    # the probabilities, and of the result; sums in fp32 are off by less than 2^-16 of all that
    p = torch.softmax(s, -1)
    e = (2.0 ** -11 * (q[0, :, 0].double()[:, None] * kd[0]).abs().sum(-1) * D ** -0.5).amax(-1)[:, None]
    room = (2 * e + 2.0 ** -10 + 2.0 ** -16) * (p[..., None] * vd[0].abs()).sum(1) + 2.0 ** -11 * want.abs() + 2.0 ** -20
    assert bool(((got.cpu().double()[0, :, 0] - want).abs() <= room).all())


def test_value_scales_far_apart():
    """Blocks of values from 2^-24 to 2^14 in fp16: a probability's product with its scale neither vanishes nor overflows, whichever block leads."""
    K = _K()
    announce("decode_attn_kv8 value scales")
    g = torch.Generator().manual_seed(3)
    H, D, P, n = 2, 64, 64, 16 * 24
    for dtype in (F16, BF16):
        for turn in (1, -1):
            ks = [torch.randn(H, n, D, generator=g).to(dtype)]
            size = torch.exp2(turn * torch.linspace(-14, 12, 24)).repeat_interleave(16)[None, :, None]
            vs = [(torch.randn(H, n, D, generator=g) * size).to(dtype)]
            cache = new_cache(1, H, D, P, 7, 6, dtype, I8, g)
            deal_pages(cache, [n], P, g)
            ref.put(cache, 0, ks[0], vs[0])
            for q_size in (0.1, 8.0):
                q = (q_size * torch.randn(1, 4, 1, D, generator=g)).to(dtype)
                # the keys of the smallest values as alike as can be to the queries: their weight is nearly all
                got = K.decode_attn_kv8(q.cuda(), to_gpu(cache), torch.tensor([n], dtype=torch.int32).cuda())
                check_attention(got, q, cache, [n], ks, vs, I8, D ** -0.5, (dtype, turn, q_size))


def test_long_and_ragged_with_wide_offsets():
    """Pools past 4 GiB with the sequence's pages at their far end, and a batch whose units outnumber and underfill the waves."""
    K = _K()
    announce("decode_attn_kv8 wide pools")
    g = torch.Generator().manual_seed(6)
    H, D, P = 2, 128, 128
    N = (1 << 32) // (H * P * D) + 40                          # 4 GiB and some: bytes of codes
    lens = [1000, 37]
    cache = new_cache(2, H, D, P, 16, 9, BF16, I8, g)
    deal_pages(cache, lens, P, g)
    ks, vs = rows_of(2, H, D, lens, BF16, g), rows_of(2, H, D, lens, BF16, g)
    dev = [torch.zeros((N,) + t.shape[1:], dtype=t.dtype, device="cuda") for t in cache[:4]] + [t.cuda() for t in cache[4:]]
    dev[6] = torch.where(dev[6] >= 0, dev[6] + (N - 16), -1)
    pack = lambda xs: torch.cat([x.transpose(0, 1) for x in xs]).cuda()  # noqa: E731
    at = torch.tensor(lens, dtype=torch.int32).cuda()
    K.kv8_pages_fill(pack(ks), pack(vs), dev, 2, 1000, at)
    assert int((dev[0][:N - 16] != 0).sum()) == 0 and int((dev[1][:N - 16] != 0).sum()) == 0
    q = torch.randn(2, 8, 1, D, generator=g).to(BF16)
    check_attention(K.decode_attn_kv8(q.cuda(), dev, at), q, cache, lens, ks, vs, I8, D ** -0.5, "wide")
    k, v = K.kv8_pages_read(dev, at, 1000)
    held = ref.Cache(H, D, I8)
    assert torch.equal(k[0].cpu(), held.held(ks[0]).float().to(BF16)) and torch.equal(v[1, :, :37].cpu(), held.held(vs[1]).float().to(BF16))


@pytest.mark.parametrize("dtype,code,Hq,H,D,B,lo,hi", [
    (F16, I8, 16, 8, 64, 3, 30000, 40000),           # shares of several tiles, taken as waves come to the end of theirs
    (BF16, E4, 40, 40, 128, 30, 0, 2100),            # several units a share
    (BF16, I8, 8, 1, 128, 1, 70001, 70001),          # hundreds of shares a unit
    (F16, E4, 34, 2, 80, 70, 1000, 1600),            # two runs of queries a key head; more sequences than lanes
])
def test_attention_shares(dtype, code, Hq, H, D, B, lo, hi):
    """Sequences cut into many shares against float64, on the GPU (the oracle on some of the heads), and the same bits again."""
    K = _K()
    announce("decode_attn_kv8 shares", dtype, code, Hq, H, D, B, lo, hi)
    g = torch.Generator().manual_seed(B + hi)
    lens = torch.randint(lo, hi + 1, (B,), generator=g).tolist()
    P = 64
    cache = list(K.kv8_pages(sum(n // P + 1 for n in lens), B, H, P, D, hi // P + 2, dtype, "cuda", code))
    table = torch.full(cache[6].shape, -1, dtype=torch.int32)
    ids = torch.randperm(cache[0].shape[0], generator=g).tolist()
    for b, n in enumerate(lens):
        for pi in range(-(-n // P)):
            table[b, pi] = ids.pop()
    cache[6] = table.cuda()
    gg = torch.Generator(device="cuda").manual_seed(1)
    kv = torch.randn(sum(lens), 2 * H, D, generator=gg, device="cuda", dtype=dtype)
    at = torch.tensor(lens, dtype=torch.int32).cuda()
    K.kv8_pages_fill(kv[:, :H], kv[:, H:], cache, B, max(lens), at)
    q = 2 * torch.randn(B, Hq, 1, D, generator=gg, device="cuda", dtype=dtype)
    got = K.decode_attn_kv8(q, cache, at)
    assert torch.equal(got, K.decode_attn_kv8(q, cache, at))
    half = torch.finfo(dtype).eps / 2
    k, v = K.kv8_pages_read(cache, at, max(lens))                       # rounded to the type: K and V again half a step off
    for b in range(0, B, max(1, B // 6)):
        n = lens[b]
        kb, vb = k[b, :, :n].double(), v[b, :, :n].double()
        qb = q[b, :, 0].double().view(H, -1, D)
        p = torch.softmax(qb @ kb.transpose(-1, -2) * D ** -0.5, -1)
        want, size = p @ vb, p @ vb.abs()
        # a key half a step off moves a score by that of sum |q k|, at most 40 here (2 x 128 products of N(0,1) / sqrt(128), by 3): in the mean it is far less,
        # and it is the root of the sum of squares that counts: sqrt(sum (q k)^2) / sqrt(D) half, under 8 half
        tol = half * (size + want.abs()) + half * size + 8 * half * size
        off = ((got[b, :, 0].double().view(want.shape) - want).abs() - tol).max()
        assert n == 0 or off <= 0, (b, n, float(off))


@pytest.mark.parametrize("seed", range(8))
def test_attention_random(seed):
    K = _K()
    g = torch.Generator().manual_seed(500 + seed)
    pick = lambda xs: xs[int(torch.randint(0, len(xs), (1,), generator=g))]  # noqa: E731
    dtype, code, D, P = pick([F16, BF16]), pick([I8, E4]), pick([16, 64, 80, 96, 112, 128]), pick([16, 32, 64, 128])
    H, G, B = pick([1, 2, 3, 8]), pick([1, 1, 2, 5, 8, 16, 17]), int(torch.randint(1, 70, (1,), generator=g))
    lens = torch.randint(0, pick([20, 300, 900]), (B,), generator=g).tolist()
    announce("decode_attn_kv8 random", seed, dtype, code, H, G, D, P, lens[:8])
    cache = new_cache(B, H, D, P, sum(n // P + 1 for n in lens) + 2, max(lens) // P + 1, dtype, code, g)
    deal_pages(cache, lens, P, g)
    ks, vs = rows_of(B, H, D, lens, dtype, g), rows_of(B, H, D, lens, dtype, g)
    pack = lambda xs: torch.cat([x.transpose(0, 1) for x in xs]).cuda()  # noqa: E731
    dev = to_gpu(cache)
    at = torch.tensor(lens, dtype=torch.int32).cuda()
    K.kv8_pages_fill(pack(ks), pack(vs), dev, B, max(lens), at)
    q = (2 * torch.randn(B, G * H, 1, D, generator=g)).to(dtype)
    few = list(range(0, B, max(1, B // 12)))
    got = K.decode_attn_kv8(q.cuda(), dev, at)
    check_attention(got[few], q[few], cache, [lens[b] for b in few], [ks[b] for b in few], [vs[b] for b in few], code, D ** -0.5, "random")
    assert bool((got[[b for b in range(B) if lens[b] == 0]] == 0).all())
    assert torch.equal(got, K.decode_attn_kv8(q.cuda(), dev, at))       # the same call, the same bits


def test_two_captured_steps_and_streams():
    """A decode step captured twice (lengths that advance in place) replays in turn with eager steps on the same caches; another stream."""
    K = _K()
    from energonai_amd.seqinfo import SeqInfo
    announce("kv8 captured")
    g = torch.Generator().manual_seed(12)
    B, Hq, H, D, P = 3, 8, 2, 64, 16
    lens = [30, 47, 3]
    cache = new_cache(B, H, D, P, 40, 8, BF16, E4, g, garbage=False)
    deal_pages(cache, [120] * B, P, g)
    ks, vs = rows_of(B, H, D, lens, BF16, g), rows_of(B, H, D, lens, BF16, g)
    for b in range(B):
        ref.put(cache, b, ks[b], vs[b])
    rot = K.rotary_table(128, D)
    x = torch.randn(B, Hq + 2 * H, D, device="cuda", dtype=BF16)

    def state():
        at = torch.tensor(lens, dtype=torch.int32).cuda()
        return to_gpu(cache), at, SeqInfo(at, None, B, None, at)

    def step(s):
        dev, at, info = s
        q = K.kv8_pages_append(x[:, :Hq], x[:, Hq:Hq + H], x[:, Hq + H:], dev, info, rot)
        at.add_(1)
        return K.decode_attn_kv8(q, dev, info)
    step(state())
    pairs = [(state(), state()) for _ in range(2)]
    graphs = []
    for captured, _ in pairs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(captured)
        captured[1].copy_(torch.tensor(lens, dtype=torch.int32))
        graphs.append((graph, out))
    for i in range(20):
        x.copy_(torch.randn(x.shape, generator=g).to(BF16))
        for graph, _ in graphs:
            graph.replay()
        for (graph, out), (captured, eager) in zip(graphs, pairs):
            want = step(eager)
            torch.cuda.synchronize()
            assert torch.equal(out, want), i
    for captured, eager in pairs:
        assert all(same_bits(a, b) for a, b in zip(captured[0], eager[0]))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    a, b = state(), state()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        on_s = step(a)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(on_s, step(b))


def test_nothing_cached():
    """No sequences, no pages, no positions, sequences of length zero between others: nothing is read, zeros come back."""
    K = _K()
    announce("kv8, nothing cached")
    H, D = 2, 64
    none = K.kv8_pages(1, 3, H, 16, D, 0, F16, "cuda")
    zero = torch.zeros(3, dtype=torch.int32, device="cuda")
    many = torch.tensor([0, 5, 1 << 30], dtype=torch.int32, device="cuda")
    q = torch.randn(3, 4, 1, D, device="cuda", dtype=F16)
    over = torch.zeros(1, dtype=torch.int32, device="cuda")
    x = torch.randn(3, H, D, device="cuda", dtype=F16)
    for lens in (zero, many):
        assert bool((K.decode_attn_kv8(q, none, lens) == 0).all())
        assert all(bool((t == 0).all()) for t in K.kv8_pages_read(none, lens, 20))
        K.kv8_pages_append(None, x, x, none, lens, overflow=over.zero_())
        assert int(over) == 3
    K.kv8_pages_fill(x, x, none, 3, 4, torch.tensor([1, 0, 2], dtype=torch.int32, device="cuda"), overflow=over.zero_())
    assert int(over) == 3 and all(bool((t == 0).all()) for t in none[:6])
    big = K.kv8_pages(4, 3, H, 16, D, 5000, F16, "cuda")              # capacity for the second form of the attention, no page, no position
    assert bool((K.decode_attn_kv8(q, big, zero) == 0).all())
    empty = K.kv8_pages(1, 0, H, 16, D, 2, F16, "cuda")
    for call in (lambda: K.decode_attn_kv8(q[:0], empty, zero[:0]), lambda: K.kv8_pages_read(empty, zero[:0], 3)):
        with pytest.raises(RuntimeError):                             # a batch of no sequences has no lengths, here as anywhere in the package
            call()
    assert K.kv8_pages_read(big, zero, 0)[0].shape == (3, H, 0, D)
    one = K.rotary_table(4, D)
    for t in K.qk_norm_rotary(x[:0], x[:0], 3, zero, one):
        assert t.shape == (0, H, D)


def test_refusals():
    K = _K()
    announce("kv8 refusals")
    B, H, D, P = 2, 2, 64, 32
    make = lambda **kw: list(K.kv8_pages(**{**dict(pool_pages=4, batch_size=B, head_num=H, page_size=P, size_per_head=D, max_pages_per_seq=2,  # noqa: E731
                                                   dtype=F16, device="cuda", code_dtype=I8), **kw}))
    good = make()
    x = torch.zeros(B, H, D, device="cuda", dtype=F16)
    q = torch.zeros(B, 4, 1, D, device="cuda", dtype=F16)
    at = torch.zeros(B, dtype=torch.int32, device="cuda")

    def calls(c, rows=x, q_=q, lens=at):
        return [lambda: K.kv8_pages_fill(rows, rows, c, B, 1, lens + 1), lambda: K.kv8_pages_append(None, rows, rows, c, lens),
                lambda: K.kv8_pages_read(c, lens, 4), lambda: K.decode_attn_kv8(q_, c, lens)]
    for call in calls(good):
        call()
    torch.cuda.synchronize()
    swaps = [(0, good[0].cpu()), (0, good[0].float()), (0, good[0].view(E4)), (0, good[0][..., :32]), (0, good[0][:0]), (0, good[0][:, :, :24]),
             (0, good[0].transpose(1, 2)), (1, good[1].view(4, H, P, D)), (1, good[1].transpose(3, 4)), (2, good[2].half()), (3, good[3][:3]),
             (4, good[4].float()), (4, good[4].to(BF16)), (4, good[4][:1]), (5, good[5].transpose(2, 3)), (6, good[6].long()), (6, good[6][:1])]
    for i, t in swaps:
        c = list(good)
        c[i] = t
        for call in calls(c):
            with pytest.raises(RuntimeError):
                call()
    for call in calls(good[:6]):
        with pytest.raises(RuntimeError):
            call()
    for rows in (x.float(), x[:, :1], x[..., :32], x.cpu(), x[0]):
        for call in calls(good, rows=rows)[:2]:
            with pytest.raises(RuntimeError):
                call()
    for bad in (q.float(), q[:1], q[:, :3], q[:, :1], q[..., :32], q.cpu(), q.view(-1)):
        with pytest.raises(RuntimeError):
            K.decode_attn_kv8(bad, good, at)
    with pytest.raises(RuntimeError):
        K.decode_attn_kv8(q, make(max_pages_per_seq=1000), at, workspace=torch.zeros(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(RuntimeError):
        K.decode_attn_kv8(q, good, at, out=q.float())
    with pytest.raises(RuntimeError):
        K.decode_attn_kv8(q, good, at[:1])
    with pytest.raises(RuntimeError):
        K.kv8_pages_read(good, at, -1)
    with pytest.raises(RuntimeError):
        K.kv8_pages_read(good, at, 4, first=at.long())
    with pytest.raises(RuntimeError):
        K.kv8_pages_fill(x, x, good, B + 1, 1, at)
    for kw in (dict(page_size=24), dict(page_size=8), dict(size_per_head=40), dict(size_per_head=144), dict(dtype=torch.float32), dict(code_dtype=torch.uint8)):
        with pytest.raises(RuntimeError):
            make(**kw)
