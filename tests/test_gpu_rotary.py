"""Norm and rotation of queries and keys, on packed rows and on the way into a paged cache, against float64."""
import pytest
import torch

from gpu_util import announce
from oracle import kv8 as ref

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _K():
    import energonai_amd.kernel as K
    return K


def assert_rows(got, want, size, dtype, what):
    """Half a step of the type, and what fp32 adds on the way: the norm's sum of up to 256 squares over lanes of at most 16 each (22
    roundings, half of them on the root), root, quotient, gain and rotation (8 more): under 32 half steps of fp32 of both channels of the pair."""
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    tol = torch.finfo(dtype).eps / 2 * want.abs() + 32 * 2.0 ** -24 * size + (2.0 ** -25 if dtype == F16 else 0.0)
    off = ((got - want).abs() - tol)[~torch.isnan(want)]
    assert off.numel() == 0 or off.max() <= 0, (what, float(off.max()))


def _projection(rows, heads, D, dtype, seed, pad=0):
    """Views ``[rows, heads_i, D]`` of one projection whose rows have ``pad`` more elements."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, sum(heads) * D + pad, generator=g).to(dtype)
    gpu = x.cuda()
    cpu_views, views, at = [], [], 0
    for h in heads:
        cpu_views.append(x[:, at:at + h * D].unflatten(1, (h, D)))
        views.append(gpu[:, at:at + h * D].unflatten(1, (h, D)))
        at += h * D
    return cpu_views, views


CASES = [
    # dtype, lens, Hq, Hk, D, R, interleaved, q gain, k gain, pad
    (F16, [1], 12, 12, 64, 64, False, False, False, 0),
    (BF16, [5, 0, 33, 1, 0], 32, 8, 128, 128, False, True, True, 0),
    (F32, [7, 40], 4, 2, 96, 48, True, True, False, 0),
    (F16, [130, 3], 5, 5, 80, 40, False, False, True, 3),            # four channels a vector; rows off every boundary
    (BF16, [19], 7, 1, 112, 28, False, True, True, 1),               # two
    (F16, [19, 19], 3, 3, 80, 20, True, False, False, 0),
    (F16, [9], 2, 3, 36, 10, False, True, True, 0),                  # one
    (F32, [9], 2, 3, 7, 6, True, True, True, 0),                     # a head of seven channels, one behind its pairs
    (BF16, [21], 3, 1, 256, 256, False, True, True, 0),
    (F32, [21], 3, 1, 256, 64, True, True, False, 0),
    (F16, [4], 2, 2, 250, 6, False, True, True, 0),                  # 125 units of one channel a side: two a lane
    (F16, [11, 6], 9, 0, 64, 64, True, True, False, 0),              # queries alone
    (BF16, [3, 4], 6, 2, 64, 0, False, True, True, 0),               # norms alone
    (F16, [900, 1, 77], 20, 4, 128, 32, True, False, False, 0),      # many rows: four heads a group, 20 and 4 of them
    (BF16, [700, 411], 13, 3, 64, 64, False, True, True, 0),         # 13 = 3 groups of four and one
]


@pytest.mark.parametrize("dtype,lens,Hq,Hk,D,R,il,qn,kn,pad", CASES)
def test_qk_norm_rotary(dtype, lens, Hq, Hk, D, R, il, qn, kn, pad):
    K = _K()
    announce("qk_norm_rotary", dtype, lens, Hq, Hk, D, R, il, qn, kn, pad)
    T = sum(lens)
    (q, k), (qd, kd) = _projection(T + 2, [Hq, Hk], D, dtype, 7 * D + R, pad)
    g = torch.Generator().manual_seed(1)
    gains = [(1 + 0.1 * torch.randn(D, generator=g)).to(dtype) if on else None for on in (qn, kn)]
    rotary = ref.table(max(lens), R) if R else None
    pos = torch.cat([torch.arange(n) for n in lens])
    lens_t = torch.tensor(lens, dtype=torch.int32).cuda()
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    kw = dict(q_weight=dev(gains[0]), k_weight=dev(gains[1]), eps=1e-5, interleaved=il)
    rot = None if rotary is None else tuple(t.cuda() for t in rotary)
    want = [ref.norm_rotary(x[:T], pos, rotary, w, 1e-5, il) for x, w in ((q, gains[0]), (k, gains[1]))]
    got = K.qk_norm_rotary(qd[:T], kd[:T] if Hk else None, len(lens), lens_t, rot, **kw)
    for y, (w, size), n, h in zip(got, want, "qk", (Hq, Hk)):
        if h:
            assert y.is_contiguous() and y.dtype == dtype
            assert_rows(y, w, size, dtype, n)
    # two rows behind the last sequence stay as they are, and the rows may be written where they were read
    out = (torch.full((T + 2, Hq, D), 7.0, dtype=dtype, device="cuda"), torch.full((T + 2, Hk, D), 7.0, dtype=dtype, device="cuda") if Hk else None)
    again = K.qk_norm_rotary(qd, kd if Hk else None, len(lens), lens_t, rot, out=out, **kw)
    for y, z in zip(again, got):
        if z is not None:
            assert torch.equal(y[:T], z) and bool((y[T:] == 7.0).all())
    place = K.qk_norm_rotary(qd, kd if Hk else None, len(lens), lens_t, rot, out=(qd, kd if Hk else None), **kw)
    assert place[0] is qd and torch.equal(qd[:T], got[0]) and torch.equal(qd[T:].cpu(), q[T:])
    if Hk:
        assert torch.equal(kd[:T], got[1]) and torch.equal(kd[T:].cpu(), k[T:])


def test_positions_given():
    """Positions in any order; one outside the table makes the rotated channels NaN and leaves the others."""
    K = _K()
    announce("qk_norm_rotary positions")
    T, H, D, R = 6, 3, 64, 32
    (q, k), (qd, kd) = _projection(T, [H, H], D, F16, 3)
    q[2, :, 40], qd[2, :, 40] = float("inf"), float("inf")           # not rotated: stays what it is, and stays alone
    cos, sin = ref.table(50, R)
    pos = torch.tensor([49, 3, 3, 50, -1, 0], dtype=torch.int32)
    got = K.qk_norm_rotary(qd, kd, 0, None, (cos.cuda(), sin.cuda()), positions=pos.cuda())
    for y, x in zip(got, (q, k)):
        y = y.cpu()
        want, size = ref.norm_rotary(x, pos.clamp(0, 49).long(), (cos, sin), None, 0.0, False)
        for t in (0, 1, 5):
            assert_rows(y[t], want[t], size[t], F16, t)
        for t in (3, 4):
            assert torch.isnan(y[t, :, :R]).all() and torch.equal(y[t, :, R:], x[t, :, R:])
    assert torch.equal(got[0][2, :, R:].cpu(), q[2, :, R:]) and torch.isfinite(got[0][2, :, :R]).all()


def test_far_positions_and_table():
    K = _K()
    announce("rotary_table")
    cos, sin = K.rotary_table(131072, 64)
    for p in (0, 1, 4097, 131071):
        for i in (0, 1, 31):
            a = p * 10000.0 ** (-2 * i / 64)
            assert abs(cos[p, i].item() - __import__("math").cos(a)) < 1e-7 and abs(sin[p, i].item() - __import__("math").sin(a)) < 1e-7
    (q, k), (qd, kd) = _projection(2, [2, 2], 64, F32, 5)
    pos = torch.tensor([131071, 100003], dtype=torch.int32)
    got = K.qk_norm_rotary(qd, kd, 0, None, (cos, sin), positions=pos.cuda(), interleaved=True)
    want, size = ref.norm_rotary(q, pos.long(), (cos.cpu(), sin.cpu()), None, 0.0, True)
    assert_rows(got[0], want, size, F32, "far")
    with pytest.raises(ValueError):
        K.rotary_table(10, 5)


@pytest.mark.parametrize("dtype,B,Hq,H,D,R,il,P,norm", [
    (F16, 1, 12, 12, 64, 64, False, 16, False), (BF16, 9, 16, 2, 128, 128, False, 64, True), (F32, 5, 6, 3, 96, 48, True, 32, True),
    (F16, 4, 3, 3, 50, 6, False, 16, True), (BF16, 70, 8, 8, 80, 80, True, 128, False),
])
def test_append_rotary(dtype, B, Hq, H, D, R, il, P, norm):
    """The bits of qk_norm_rotary at the lengths, in their pages, and nothing else written; a sequence without a page is counted, its query turned all the same."""
    K = _K()
    announce("kv_pages_append_rotary", dtype, B, Hq, H, D, R, il, P, norm)
    g = torch.Generator().manual_seed(B + D)
    lens = torch.randint(0, 5 * P, (B,), generator=g, dtype=torch.int32)
    lens[0] = 2 * P - 1
    _, (q, k, v) = _projection(B, [Hq, H, H], D, dtype, D, 5)
    gains = [(1 + 0.1 * torch.randn(D, generator=g)).to(dtype).cuda() if norm else None for _ in range(2)]
    rot = K.rotary_table(5 * P, R)
    N = B * 5 + 2
    table = torch.randperm(N, generator=g)[:B * 5].view(B, 5).to(torch.int32).cuda()
    if B > 3:
        table[1, int(lens[1]) // P] = N
        table[2, int(lens[2]) // P] = -1
    lost = 2 if B > 3 else 0
    pool = torch.randn(N, 2, H, P, D, generator=g).to(dtype).cuda()
    want_pool = pool.clone()
    at = lens.cuda()
    over = torch.zeros(1, dtype=torch.int32, device="cuda")
    kw = dict(q_weight=gains[0], k_weight=gains[1], interleaved=il)
    want_q, turned = K.qk_norm_rotary(q, k, B, None, rot, positions=at, **kw)
    for b in range(B):
        n = int(lens[b])
        pid = int(table[b, n // P])
        if 0 <= pid < N:
            want_pool[pid, 0, :, n % P], want_pool[pid, 1, :, n % P] = turned[b], v[b]
    for again in range(2):                               # the same again changes nothing
        got = K.kv_pages_append_rotary(q, k, v, pool[:, 0], pool[:, 1], at, table, rot, overflow=over.zero_(), **kw)
        assert torch.equal(got, want_q) and torch.equal(pool, want_pool) and int(over) == lost


def test_captured_and_on_another_stream():
    """A captured call replays on new rows in the same tensors; a call on another stream does its work there."""
    K = _K()
    from energonai_amd.seqinfo import build_seq_info
    announce("rotary captured")
    lens = torch.tensor([40, 3, 17], dtype=torch.int32, device="cuda")
    info = build_seq_info(lens, 3)
    _, (q, k) = _projection(60, [8, 2], 64, BF16, 1)
    rot = K.rotary_table(64, 64)
    pool = torch.zeros(2, 4, 2, 16, 64, device="cuda", dtype=BF16)
    table = torch.arange(3, dtype=torch.int32, device="cuda").view(3, 1)
    at = torch.tensor([3, 9, 15], dtype=torch.int32, device="cuda")
    from energonai_amd.seqinfo import SeqInfo
    ainfo = SeqInfo(at, None, 3, None, at)

    def step():
        a = K.qk_norm_rotary(q, k, 3, info, rot)
        return a + (K.kv_pages_append_rotary(q[:3], k[:3], k[3:6], pool[0], pool[1], ainfo, table, rot),)
    step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        on_s = step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(3):
        fresh = torch.randn_like(q)
        q.copy_(fresh)
        pool.zero_()
        graph.replay()
        torch.cuda.synchronize()
        kept = pool.clone()
        pool.zero_()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(held, want)) and torch.equal(pool, kept)
    assert on_s[0].shape == (60, 8, 64)


def test_refusals():
    K = _K()
    announce("rotary refusals")
    lens = torch.tensor([4], dtype=torch.int32, device="cuda")
    x = torch.zeros(4, 2, 64, device="cuda", dtype=F16)
    rot = K.rotary_table(8, 64)
    ok = lambda **kw: K.qk_norm_rotary(*[kw.pop(n, d) for n, d in (("q", x), ("k", x), ("B", 1), ("lens", lens), ("rot", rot))], **kw)  # noqa: E731
    ok()
    from energonai_amd.seqinfo import SeqInfo, build_seq_info
    both = torch.zeros(4, 4, 64, device="cuda", dtype=F16)
    ok(q=both[:, :2], k=both[:, 2:], out=(both[:, :2], both[:, 2:]))          # two views of one projection, each over itself
    y = torch.zeros(4, 2, 64, device="cuda", dtype=F16)
    for out in ((y, x), (y, x[:, :1].expand(4, 2, 64)), (y, y), (torch.zeros(2, 64, device="cuda", dtype=F16).expand(4, 2, 64), y), (x[:, 1:].expand(4, 2, 64), y)):
        with pytest.raises(RuntimeError):
            ok(q=x, k=torch.ones_like(x), out=out)
    with pytest.raises(RuntimeError):
        ok(q=both[:, :2], k=both[:, 2:], out=(both[:, 2:], both[:, :2]))       # each over the other
    for bad in (dict(q=x.cpu()), dict(q=x.float()), dict(q=x.to(torch.float64), k=None), dict(k=x[:3]), dict(k=x[..., :32]), dict(q=x.transpose(1, 2)),
                dict(q=x[0]), dict(rot=(rot[0].half(), rot[1])), dict(rot=(rot[0], rot[1][:4])), dict(rot=K.rotary_table(8, 66)), dict(rot=(rot[0].cpu(), rot[1])),
                dict(rot=(rot[0][:0], rot[1][:0])), dict(rot=(rot[0][:, :0].contiguous(), rot[1][:, :0].contiguous())),
                dict(rot=(rot[0][:, :0].contiguous(), rot[1][:, :0].contiguous()), lens=build_seq_info(lens, 1)), dict(q_weight=torch.ones(64, device="cuda")), dict(k_weight=torch.ones(32, device="cuda", dtype=F16)),
                dict(out=(x,)), dict(out=(x, x.float())), dict(positions=torch.zeros(3, dtype=torch.int32, device="cuda")),
                dict(positions=torch.zeros(4, dtype=torch.int64, device="cuda")), dict(lens=SeqInfo(lens, None, 1, None, lens)),
                dict(q=torch.zeros(4, 2, 257, device="cuda", dtype=F16), k=None, rot=None)):
        with pytest.raises(RuntimeError):
            ok(**bad)
    pool = torch.zeros(2, 3, 2, 16, 64, device="cuda", dtype=F16)
    table = torch.zeros(4, 1, dtype=torch.int32, device="cuda")
    at = torch.zeros(4, dtype=torch.int32, device="cuda")
    args = dict(q=x, k=x, v=x, kp=pool[0], vp=pool[1], lens=at, table=table, rot=rot)
    call = lambda **kw: K.kv_pages_append_rotary(*{**args, **kw}.values())  # noqa: E731
    call()
    for bad in (dict(q=x[:3]), dict(k=x[:, :1]), dict(v=x.float()), dict(kp=pool[0].float()), dict(vp=pool[1][..., :32]), dict(table=table.long()),
                dict(table=table[:3]), dict(lens=at[:3]), dict(q=None), dict(rot=K.rotary_table(8, 66)), dict(kp=pool[0][:, :, :8], vp=pool[1][:, :, :8])):
        with pytest.raises(RuntimeError):
            call(**bad)
