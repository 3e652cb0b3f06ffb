"""Decode steps of drafted tokens over a paged cache against a plain restatement in 64 bits: trees, their attention, acceptance, and the
accepted rows' way into the cache."""
import random

import pytest
import torch

from gpu_util import announce
from oracle import drafts as ref

pytestmark = pytest.mark.gpu


def K():
    from energonai_amd import kernel
    return kernel


def trees(counts, seed, reach=4):
    r = random.Random(seed)
    return [p for n in counts for p in [-1][:n] + [r.randint(max(0, i - reach), i - 1) for i in range(1, n)]]


def step(lens, counts, Hq, H, D, P, dtype, seed, extra_pages=2, table_pages=None):
    """A batch on the CPU: queries, new rows, pools with NaN in all that is no cached position, a table in any order."""
    g = torch.Generator().manual_seed(seed)
    held = [-(-(n + m) // P) for n, m in zip(lens, counts)]
    N, width = sum(held) + extra_pages, max(max(held), 1) if table_pages is None else table_pages
    ids = torch.randperm(N, generator=g, dtype=torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    pools = [torch.full((N, H, P, D), float("nan"), dtype=dtype) for _ in range(2)]
    at = 0
    for b, n in enumerate(lens):
        table[b, :held[b]] = ids[at:at + held[b]]
        at += held[b]
        for pool in pools:
            rows = torch.randn(n, H, D, generator=g).to(dtype)
            for j in range(0, n, P):
                pool[table[b, j // P], :, :min(P, n - j)] = rows[j:j + P].transpose(0, 1)
    T = sum(counts)
    q, k, v = (torch.randn(T, h, D, generator=g).mul(1.5 if h == Hq and i == 0 else 1).to(dtype) for i, h in enumerate((Hq, H, H)))
    return q, k, v, pools[0], pools[1], table


def tolerance(want, size, most, dtype, D, keys):
    """Half a step of the result and of every probability (sum p |v| / sum p of them); a score's fp32 sum of D products and its scaling,
    each (D + 4) halves of 2^-23 of sum |q k| scale, in the numerator and the sum; the fp32 sums over the keys; in fp16 a probability below 2^-14
    is off by 2^-25 of the largest, and values are below 8."""
    half = torch.finfo(dtype).eps / 2
    fp32 = size * (2 * most * (D + 4) * 2 ** -24 + 2 * (keys + 16) * 2 ** -24)
    return half * want.abs() + half * size + fp32 + (keys * 2 ** -25 * 8 if dtype == torch.float16 else 0) + 1e-30


def run(q, k, v, kp, vp, lens, table, tree, **kw):
    cuda = lambda t: t.cuda()  # noqa: E731
    return K().decode_attn_tree(cuda(q), cuda(k), cuda(v), cuda(kp), cuda(vp), torch.tensor(lens, dtype=torch.int32, device="cuda"), cuda(table), tree, **kw).cpu()


CASES = [
    # lens, counts, Hq, H, D, P
    ([0], [1], 1, 1, 64, 16),
    ([1], [1], 2, 2, 64, 16),
    ([100], [8], 12, 12, 64, 16),
    ([63, 64, 65, 0], [1, 2, 3, 4], 4, 2, 128, 64),
    ([127, 128, 129], [16, 15, 17], 4, 4, 128, 32),
    ([700, 0, 3], [64, 63, 64], 3, 3, 64, 64),
    ([250, 40], [64, 7], 8, 1, 128, 16),
    ([33, 500], [5, 0], 16, 1, 96, 64),
    ([90, 17, 300], [0, 0, 9], 10, 5, 80, 128),
    ([77, 200], [12, 30], 14, 2, 112, 16),
    ([31, 130], [6, 20], 6, 3, 72, 32),
    ([31, 130], [6, 20], 6, 3, 8, 16),
    ([257], [33], 5, 5, 24, 16),
    ([1500], [2], 8, 8, 40, 64),
    ([2000, 1], [16, 64], 7, 1, 128, 64),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,counts,Hq,H,D,P", CASES)
def test_attention(lens, counts, Hq, H, D, P, dtype):
    announce("tree attention", lens, counts, Hq, H, D, P, dtype)
    q, k, v, kp, vp, table = step(lens, counts, Hq, H, D, P, dtype, len(lens) * 1000 + D)
    parents = trees(counts, D + P)
    tree = K().draft_tree(torch.tensor(parents, dtype=torch.int32, device="cuda"), counts, len(counts), max(max(counts), 1))
    masks, depths = ref.masks(parents, counts)
    assert tree.masks.tolist() == masks and tree.depths.tolist() == depths
    want, size, most = ref.attend(q, k, v, kp, vp, lens, table, masks, counts)
    got = run(q, k, v, kp, vp, lens, table, tree)
    off = (got.double() - want).abs() - tolerance(want, size, most, dtype, D, max(lens) + 64)
    assert float(off.max()) <= 0, float(off.max())


@pytest.mark.parametrize("B,H,Hq,longest,most", [(70, 2, 4, 700, 5), (150, 3, 3, 1300, 2), (130, 1, 17, 600, 9)])
def test_batches_of_more_than_a_wave_of_sequences(B, H, Hq, longest, most):
    """Runs of tiles over many sequences, among them ones without nodes, without positions, without either."""
    r = random.Random(B)
    counts = [r.choice([0, 1, most]) for _ in range(B - 1)] + [most]
    lens = [r.choice([0, 1, 63, 64, r.randrange(200)]) for _ in range(B - 1)] + [longest - most]
    counts[:2] = counts[66:68] = [0, 0]
    D, P, dtype = 32, 64, torch.float16
    announce("many sequences", B, H, Hq, longest, most)
    q, k, v, kp, vp, table = step(lens, counts, Hq, H, D, P, dtype, B, table_pages=21)
    assert K().decode_attn_tree_workspace_bytes(B, Hq, H, 21 * P, D, most) > 0
    parents = trees(counts, B)
    tree = K().draft_tree(torch.tensor(parents, dtype=torch.int32, device="cuda"), counts, B, most)
    masks, _ = ref.masks(parents, counts)
    want, size, top = ref.attend(q, k, v, kp, vp, lens, table, masks, counts)
    got = run(q, k, v, kp, vp, lens, table, tree)
    assert float(((got.double() - want).abs() - tolerance(want, size, top, dtype, D, longest + 64)).max()) <= 0


def test_tables_without_pages():
    """Sequences that hold nothing, in a table of no columns: the nodes see one another, and nothing has room."""
    counts, H, D, P, dtype = [3, 1], 2, 64, 16, torch.bfloat16
    q, k, v, kp, vp, _ = step([0, 0], counts, H, H, D, P, dtype, 3)
    table = torch.empty(2, 0, dtype=torch.int32)
    tree = K().draft_tree(torch.tensor([-1, 0, 0, -1], dtype=torch.int32, device="cuda"), counts, 2, 3)
    announce("tables without pages")
    for lens in ([0, 0], [5, 0]):                        # a length without pages counts as none
        want, size, most = ref.attend(q, k, v, kp, vp, [0, 0], table, ref.masks([-1, 0, 0, -1], counts)[0], counts)
        got = run(q, k, v, kp, vp, lens, table, tree)
        assert float(((got.double() - want).abs() - tolerance(want, size, most, dtype, D, 64)).max()) <= 0
    lost = torch.zeros(1, dtype=torch.int32, device="cuda")
    kp_d, vp_d = torch.ones_like(kp).cuda(), torch.ones_like(vp).cuda()
    path, taken = torch.tensor([[0, 1], [0, -1]], dtype=torch.int32, device="cuda"), torch.tensor([2, 1], dtype=torch.int32, device="cuda")
    K().kv_pages_extend(k.cuda(), v.cuda(), kp_d, vp_d, torch.zeros(2, dtype=torch.int32, device="cuda"), table.cuda(), tree, path, taken, overflow=lost)
    assert int(lost) == 3 and (kp_d == 1).all() and (vp_d == 1).all()


@pytest.mark.parametrize("counts,most", [([20, 64, 5], 6), ([70, 3], 64), ([1, 2], 64)])
def test_nodes_past_the_largest_do_not_exist(counts, most):
    """Rows behind ``max_nodes`` nodes of a sequence keep what is in them, and no other node sees them."""
    lens, Hq, H, D, P, dtype = [30, 7, 100][:len(counts)], 4, 2, 64, 16, torch.float16
    q, k, v, kp, vp, table = step(lens, counts, Hq, H, D, P, dtype, most)
    parents = trees(counts, most)
    tree = K().draft_tree(torch.tensor(parents, dtype=torch.int32, device="cuda"), counts, len(counts), most)
    masks, first, there = ref.masks(parents, counts)[0], 0, []
    for n in counts:
        there += [i < most for i in range(n)]
        first += n
    masks = [m & ((1 << most) - 1) if most < 64 else m for m in masks]
    want, size, top = ref.attend(q, k, v, kp, vp, lens, table, masks, counts)
    announce("nodes past the largest", counts, most)
    out = torch.full((len(parents), Hq, D), 9.0, dtype=dtype, device="cuda")
    got = run(q, k, v, kp, vp, lens, table, tree, out=out)
    there = torch.tensor(there)
    off = ((got.double() - want).abs() - tolerance(want, size, top, dtype, D, 164))[there]
    assert float(off.max()) <= 0 and (got[~there] == 9).all()


def test_pools_past_4_gib():
    """Pages whose offsets pass 32 bits, read and written."""
    H, D, P, dtype, counts, lens = 8, 128, 128, torch.float16, [3, 2], [300, 90]
    N = (5 << 30) // (H * P * D * 2)
    q, k, v, kp, vp, table = step(lens, counts, H, H, D, P, dtype, 4)
    n = kp.shape[0]
    parents = trees(counts, 1)
    tree = K().draft_tree(torch.tensor(parents, dtype=torch.int32, device="cuda"), counts, 2, 3)
    announce("pools past 4 GiB")
    want = run(q, k, v, kp, vp, lens, table, tree)
    pools = [torch.empty((N, H, P, D), dtype=dtype, device="cuda") for _ in range(2)]
    for pool, small in zip(pools, (kp, vp)):
        pool[N - n:].copy_(small)
    far = torch.where(table >= 0, table + (N - n), table)
    lens_d = torch.tensor(lens, dtype=torch.int32, device="cuda")
    assert torch.equal(K().decode_attn_tree(q.cuda(), k.cuda(), v.cuda(), *pools, lens_d, far.cuda(), tree).cpu(), want)
    path, taken = torch.tensor([[0, 1, 2], [0, 1, -1]], dtype=torch.int32, device="cuda"), torch.tensor([3, 2], dtype=torch.int32, device="cuda")
    K().kv_pages_extend(k.cuda(), v.cuda(), *pools, lens_d, far.cuda(), tree, path, taken)
    for pool, small, new in zip(pools, (kp, vp), (k, v)):
        assert torch.equal(pool[N - n:].cpu().nan_to_num(), ref.extend(small, new, lens, table, counts, path.cpu(), taken.cpu())[0].nan_to_num())


def test_logits_past_4_gib():
    """Rows of logits whose offsets pass 32 bits: the way of the last trees."""
    B, n, V = 270, 64, 130000
    logits = torch.zeros(B * n, V, dtype=torch.bfloat16, device="cuda")
    assert logits.numel() * 2 > 1 << 32
    parents = ([-1] + list(range(n - 1))) * B
    tokens = torch.zeros(B * n, dtype=torch.int64)
    for b in (0, B - 1):
        for i in range(4):
            logits[b * n + i, V - 1 - i] = 1
            tokens[b * n + i + 1] = V - 1 - i
    tokens[[n * b + 1 for b in range(1, B - 1)]] = 5           # not what their roots choose, the first of equal ones
    tokens[[5, (B - 1) * n + 5]] = 1
    announce("logits past 4 GiB")
    tree = K().draft_tree(torch.tensor(parents, dtype=torch.int32, device="cuda"), [n] * B, B, n)
    path, taken, following = (t.tolist() for t in K().accept_drafts(logits, tokens.cuda(), tree))
    for b in range(B):
        m = 5 if b in (0, B - 1) else 1
        assert path[b] == list(range(m)) + [-1] * (n - m) and taken[b] == m and following[b] == 0


@pytest.mark.parametrize("counts,reach", [([64], 64), ([64, 1, 0, 5], 1), ([70, 3], 3), ([1] * 40, 1)])
def test_trees(counts, reach):
    announce("trees", counts)
    parents = trees(counts, 5, reach)
    if counts[0] == 64:
        parents[9], parents[20], parents[33] = 9, 40, -7        # no earlier node of the sequence
    tree = K().draft_tree(torch.tensor(parents, dtype=torch.int32, device="cuda"), torch.tensor(counts, device="cuda"), len(counts))
    masks, depths = ref.masks(parents, counts)
    assert tree.masks.tolist() == masks and tree.depths.tolist() == depths and tree.max_nodes == 64


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("Hq,H,D", [(4, 2, 64), (16, 2, 128), (40, 2, 64)])
def test_any_masks(Hq, H, D, dtype):
    """Masks that are no tree's, with bits of nodes that do not exist; one that sees nothing at all; a page that is none."""
    lens, counts, P = [70, 0, 40, 200], [9, 6, 64, 33], 16
    q, k, v, kp, vp, table = step(lens, counts, Hq, H, D, P, dtype, 11)
    table[0, 1] = -1
    table[3, 2] = kp.shape[0] + 5
    r = random.Random(3)
    masks = [r.getrandbits(64) - (1 << 63) for _ in range(sum(counts))]
    masks[9] = 0                                        # the second sequence has no context: an empty row
    masks[10] = -64                                     # ... and this one sees only nodes that do not exist
    tree = K().draft_tree(torch.zeros(sum(counts), dtype=torch.int32, device="cuda"), counts, 4)._replace(masks=torch.tensor(masks, device="cuda"))
    announce("any masks", Hq, H, D, dtype)
    valid, first = [], 0
    for n in counts:
        valid += [m & (1 << n) - 1 for m in masks[first:first + n]]
        first += n
    want, size, most = ref.attend(q, k, v, kp, vp, lens, table, valid, counts)
    got = run(q, k, v, kp, vp, lens, table, tree)
    assert (got[9] == 0).all() and (got[10] == 0).all()
    off = (got.double() - want).abs() - tolerance(want, size, most, dtype, D, max(lens) + 64)
    assert float(off.max()) <= 0, float(off.max())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("Hq,H", [(2, 2), (8, 1), (24, 1)])
def test_what_is_not_a_number_reaches_who_sees_it(Hq, H, dtype):
    """Not a number in a node's key or value: the nodes that see it, and no others; infinite values likewise."""
    lens, counts, D = [50, 20], [12, 6], 64
    q, k, v, kp, vp, table = step(lens, counts, Hq, H, D, 16, dtype, 21)
    parents = [-1, 0, 0, 1, 1, 2, 2, 3, 4, 5, 6, 7] + [-1, 0, 1, 2, 3, 4]
    masks, _ = ref.masks(parents, counts)
    tree = K().draft_tree(torch.tensor(parents, dtype=torch.int32, device="cuda"), counts, 2)
    clean = run(q, k, v, kp, vp, lens, table, tree)
    k[1, :, 5] = float("nan")
    v[2, :, 7] = float("inf")
    v[5, :, 0] = float("nan")
    announce("not a number", Hq, H, dtype)
    got = run(q, k, v, kp, vp, lens, table, tree)
    for i, m in enumerate(masks):
        if i >= 12 or not m & (1 << 1 | 1 << 2 | 1 << 5):
            assert torch.equal(got[i], clean[i]), i
        elif m >> 1 & 1:
            assert got[i].isnan().all(), i
        else:
            inf = torch.zeros(D, dtype=torch.bool)
            inf[7] = True
            assert (got[i][:, 7] == float("inf")).all(), i
            if m >> 5 & 1:
                assert got[i][:, 0].isnan().all()
                inf[0] = True
            assert torch.equal(got[i][:, ~inf], clean[i][:, ~inf])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_large_scores(dtype):
    """Scores that climb by far more than the exponent's room from tile to tile, and a last tile far below the first."""
    lens, counts, D, P = [600], [20], 64, 64
    q, k, v, kp, vp, table = step(lens, counts, 2, 2, D, P, dtype, 31)
    for j in range(10):
        kp[table[0, j]] *= 4 * j if j < 8 else 0.01
    parents = trees(counts, 1)
    tree = K().draft_tree(torch.tensor(parents, dtype=torch.int32, device="cuda"), counts, 1)
    want, size, most = ref.attend(q, k, v, kp, vp, lens, table, ref.masks(parents, counts)[0], counts)
    announce("large scores", dtype)
    off = (run(q, k, v, kp, vp, lens, table, tree).double() - want).abs() - tolerance(want, size, most, dtype, D, 700)
    assert float(off.max()) <= 0, float(off.max())


def test_views_outputs_and_streams():
    """Rows of a fused projection, odd strides and addresses that are copied, pools by strides, a result in place of the queries, another
    stream, a scale, lengths as a SeqInfo; rows behind the last sequence stay as they are."""
    from energonai_amd.seqinfo import build_seq_info
    lens, counts, H, D, P, dtype = [130, 40], [7, 9], 4, 64, 16, torch.float16
    q, k, v, kp, vp, table = step(lens, counts, H, H, D, P, dtype, 41)
    parents = trees(counts, 2)
    tree = K().draft_tree(torch.tensor(parents, dtype=torch.int32, device="cuda"), counts, 2)
    want = run(q, k, v, kp, vp, lens, table, tree, scale=0.3)
    info = build_seq_info(lens, 2)
    fused = torch.cat((q, k, v), 1).cuda()
    pool = torch.zeros(kp.shape[0], 2, P, H, D, dtype=dtype, device="cuda")
    pool[:, 0], pool[:, 1] = kp.transpose(1, 2).cuda(), vp.transpose(1, 2).cuda()
    kp_v, vp_v, table_d = pool[:, 0].transpose(1, 2), pool[:, 1].transpose(1, 2), table.cuda()
    announce("views")
    got = K().decode_attn_tree(fused[:, :H], fused[:, H:2 * H], fused[:, 2 * H:], kp_v, vp_v, info, table_d, tree, scale=0.3)
    assert torch.equal(got.cpu(), want)
    odd = torch.zeros(16, 3 * H, D + 2, dtype=dtype, device="cuda")[:, :, 1:-1]
    odd.copy_(fused)
    got = K().decode_attn_tree(odd[:, :H], odd[:, H:2 * H], odd[:, 2 * H:], kp_v, vp_v, info, table_d, tree, scale=0.3)
    assert torch.equal(got.cpu(), want)
    other = torch.cuda.Stream()
    q_d = q.cuda()
    torch.cuda.synchronize()
    with torch.cuda.stream(other):
        got = K().decode_attn_tree(q_d, fused[:, H:2 * H], fused[:, 2 * H:], kp_v, vp_v, info, table_d, tree, scale=0.3, out=q_d)
    other.synchronize()
    assert got.data_ptr() == q_d.data_ptr() and torch.equal(got.cpu(), want)
    # three rows more than the sequences have
    pad = torch.full((3, 3 * H, D), float("nan"), dtype=dtype, device="cuda")
    longer = torch.cat((fused, pad))
    tree3 = tree._replace(masks=torch.cat((tree.masks, tree.masks[:3])))
    out = torch.full((19, H, D), 5.0, dtype=dtype, device="cuda")
    K().decode_attn_tree(longer[:, :H], longer[:, H:2 * H], longer[:, 2 * H:], kp_v, vp_v, info, table_d, tree3, scale=0.3, out=out)
    assert torch.equal(out[:16].cpu(), want) and (out[16:] == 5).all()
    for bad in (dict(out=fused[:, H:2 * H]), dict(out=torch.empty(16, H, D, device="cuda")), dict(scale=-1.0)):
        with pytest.raises(RuntimeError):
            K().decode_attn_tree(q_d, fused[:, H:2 * H], fused[:, 2 * H:], kp_v, vp_v, info, table_d, tree, **bad)
    k_d = fused[:, H:2 * H].contiguous()
    for args in ((q_d.float(), k_d, k_d), (q_d[:, :3], k_d, k_d), (q_d, k_d[:5], k_d), (q_d, k_d, k_d.bfloat16()), (q_d[..., :60], k_d, k_d)):
        with pytest.raises(RuntimeError):
            K().decode_attn_tree(*args, kp_v, vp_v, info, table_d, tree)
    with pytest.raises(RuntimeError):
        K().decode_attn_tree(q_d, k_d, k_d, kp_v, vp_v, info, table_d, tree._replace(masks=tree.masks[:5]))
    with pytest.raises(RuntimeError):
        K().decode_attn_tree(q_d, k_d, k_d, kp_v, vp_v, build_seq_info([1, 2, 3], 3), table_d, tree)


def test_attention_of_one_node_is_the_decode_step():
    """A tree of one node over a cache that ends before it: ``decode_attn_paged`` once the node's row is in the cache."""
    lens, counts, H, D, P, dtype = [40, 200, 1], [1, 1, 1], 6, 64, 32, torch.bfloat16
    q, k, v, kp, vp, table = step(lens, counts, H, H, D, P, dtype, 51)
    tree = K().draft_tree(torch.full((3,), -1, dtype=torch.int32, device="cuda"), counts, 3, 1)
    announce("one node")
    got = run(q, k, v, kp, vp, lens, table, tree)
    kp_d, vp_d, table_d = kp.cuda(), vp.cuda(), table.cuda()
    now = torch.tensor(lens, dtype=torch.int32, device="cuda")
    K().kv_pages_append(k.cuda(), v.cuda(), kp_d, vp_d, now, table_d)
    want = K().decode_attn_paged(q.cuda().view(3, H, 1, D), kp_d, vp_d, now + 1, table_d).view(3, H, D).cpu()
    # both round their result and their probabilities
    assert ((got.double() - want.double()).abs() <= 2 ** -8 * (2 * want.double().abs() + 2)).all()


# ---- acceptance ----------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("counts,vocab", [([1], 1), ([1, 2], 7), ([24], 50257), ([64, 1, 0, 30], 5003), ([5] * 70, 1000), ([64], 130001), ([8, 3], 4096)])
def test_acceptance(counts, vocab, dtype):
    g = torch.Generator().manual_seed(vocab + len(counts))
    T = sum(counts)
    parents = trees(counts, vocab, 2)
    tokens = torch.randint(0, vocab, (T,), generator=g)
    logits = torch.randn(T, vocab, generator=g).to(dtype)
    first = 0
    for n in counts:
        for i in range(1, n):
            if random.Random(first + i).random() < 0.8:
                logits[first + parents[first + i], tokens[first + i]] = 9.0       # several children of a node may tie
        first += n
    want = ref.accept(logits, tokens.tolist(), parents, counts, max(counts))
    for ints in (torch.int64, torch.int32):
        announce("acceptance", counts, vocab, dtype, ints)
        tree = K().draft_tree(torch.tensor(parents, dtype=torch.int32, device="cuda"), counts, len(counts), max(counts))
        got = K().accept_drafts(logits.cuda(), tokens.to(ints).cuda(), tree)
        for a, b in zip(got, want):
            assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_acceptance_of_odd_logits(dtype):
    """Equal logits, zeros of both signs, infinities, NaN; rows of a wider tensor at odd addresses; repeated tokens."""
    V, counts = 999, [6, 3, 3, 3, 2]
    wide = torch.full((17, V + 8), 50.0).to(dtype)
    logits = wide[:, 3:3 + V]
    logits[:] = -1.0
    parents = [-1, 0, 0, 0, 2, 4] + [-1, 0, 1] * 3 + [-1, 0]
    tokens = torch.tensor([0, 5, 7, 7, 9, 9] + [0, 3, 4] * 3 + [1, 998])
    logits[0, 7], logits[0, 8] = 2.0, 2.0                   # the lower index; the lower of two children with that token
    logits[2, 9] = 0.0
    logits[2, 4] = -0.0                                     # equal: 4, which no child has
    logits[6, 3], logits[7, 700] = float("inf"), float("nan")
    logits[9] = float("-inf")                               # all equal: index 0
    logits[12, 3], logits[12, 900], logits[12, 901] = float("inf"), float("nan"), float("nan")
    logits[15, 998] = 0.5
    announce("odd logits", dtype)
    device = torch.full((17, V + 8), 50.0, dtype=dtype, device="cuda")
    device.copy_(wide)
    tree = K().draft_tree(torch.tensor(parents, dtype=torch.int32, device="cuda"), counts, 5, 6)
    got = K().accept_drafts(device[:, 3:3 + V], tokens.cuda(), tree)
    want = ref.accept(logits, tokens.tolist(), parents, counts, 6)
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b)
    assert got[2].tolist() == [4, 700, 0, 900, 0]


def test_acceptance_refuses():
    tree = K().draft_tree(torch.tensor([-1, 0], dtype=torch.int32, device="cuda"), [2], 1)
    logits, tokens = torch.zeros(2, 5, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    for args in ((logits.double(), tokens, tree), (logits.t(), tokens, tree), (logits, tokens[:1], tree), (logits, tokens.float(), tree), (logits[:1], tokens[:1], tree),
                 (logits, tokens, tuple(tree)), (logits, tokens, tree._replace(max_nodes=0)), (logits, tokens, tree._replace(max_nodes=65))):
        with pytest.raises(RuntimeError):
            K().accept_drafts(*args)


# ---- accepted rows ---------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H,D,P", [(12, 64, 16), (2, 128, 64), (3, 5, 16), (1, 80, 128), (2, 600, 16)])
def test_extension(H, D, P, dtype):
    lens, counts = [16, 0, 31, 95, 700, 15], [5, 9, 4, 64, 3, 1]
    q, k, v, kp, vp, table = step(lens, counts, H, H, D, P, dtype, D)
    for pool in (kp, vp):
        pool.nan_to_num_(7.0)
    path = torch.full((6, 12), -1, dtype=torch.int32)
    for b, way in enumerate(([0, 2, 4], [0], [0, 1, 2, 3], [0, 1, 5, 9, 20, 33, 63, 40, 2, 2, 3, 3], [0, 99, 1], [0, -1])):
        path[b, :len(way)] = torch.tensor(way, dtype=torch.int32)
    taken = torch.tensor([3, 1, 4, 20, 3, 2], dtype=torch.int32)
    table[3, (95 + 4) // P:] = -1                       # no room from there on
    tree = K().draft_tree(torch.tensor(trees(counts, 1), dtype=torch.int32, device="cuda"), counts, 6)
    lost = torch.zeros(1, dtype=torch.int32, device="cuda")
    (want_k, lost_k), (want_v, _) = (ref.extend(pool, new, lens, table, counts, path, taken) for pool, new in ((kp, k), (vp, v)))
    kp_d, vp_d = kp.cuda(), vp.cuda()
    both = torch.cat((k, v), 1).cuda()
    announce("extension", H, D, P, dtype)
    K().kv_pages_extend(both[:, :H], both[:, H:], kp_d, vp_d, torch.tensor(lens, dtype=torch.int32, device="cuda"), table.cuda(), tree, path.cuda(), taken.cuda(), overflow=lost)
    assert torch.equal(kp_d.cpu(), want_k) and torch.equal(vp_d.cpu(), want_v) and int(lost) == lost_k
    for bad in (dict(path=path.cuda().long()), dict(counts=taken.cuda()[:3]), dict(k_new=both[:, :H, :-1]), dict(k_new=both[:5, :H]), dict(overflow=lost.float())):
        args = {**dict(k_new=both[:, :H], v_new=both[:, H:], k_pool=kp_d, v_pool=vp_d, kv_len_list=lens, page_table=table.cuda(), tree=tree, path=path.cuda(), counts=taken.cuda()), **bad}
        with pytest.raises(RuntimeError):
            K().kv_pages_extend(**args)


# ---- together ----------------------------------------------------------------------------------------------------------------------------


def _drafted(greedy, counts, parents, vocab, seed):
    """Tokens of the nodes: the root's is the newest; of the others some are what greedy decoding would choose."""
    r = random.Random(seed)
    tokens, first = [], 0
    for b, n in enumerate(counts):
        for i in range(n):
            tokens.append(greedy[b][0] if i == 0 else r.choice([greedy[b][min(len(greedy[b]) - 1, _depth(parents, first, i))], r.randrange(vocab)]))
        first += n
    return tokens


def _depth(parents, first, i):
    d = 0
    while parents[first + i] >= 0:
        i = parents[first + i]
        d += 1
    return d


@pytest.mark.parametrize("graph", [False, True])
def test_steps_together_decode_what_single_tokens_do(graph):
    """A small model of one layer (embedding, 4-bit projection, rotation by position, attention, 4-bit logits): some steps of drafted trees
    give the tokens and the cache that steps of one token give, eagerly and as a replayed graph."""
    from energonai_amd.seqinfo import SeqInfo, build_seq_info
    k4, dtype, B, H, D, P, V = K(), torch.float16, 3, 4, 64, 16, 211
    hid, counts = H * D, [9, 6, 12]
    g = torch.Generator(device="cuda").manual_seed(7)
    embed = torch.randn(V, hid, generator=g, device="cuda", dtype=dtype)
    qkv = k4.w4_quantize((torch.randn(3 * hid, hid, generator=g, device="cuda") / hid ** 0.5).to(dtype), 64)
    head = k4.w4_quantize((torch.randn(V, hid, generator=g, device="cuda") / hid ** 0.5).to(dtype), 32, True)
    rotary, T, steps = k4.rotary_table(400, D), sum(counts), 5
    parents = trees(counts, 9, 3)
    start = [40, 1, 75]
    table = torch.arange(B * 16, dtype=torch.int32, device="cuda").view(B, 16)
    context = [torch.randn(B * 16, H, P, D, generator=g, device="cuda", dtype=dtype) for _ in range(2)]
    tree = k4.draft_tree(torch.tensor(parents, dtype=torch.int32, device="cuda"), build_seq_info(counts, B), B, 12)
    one = k4.draft_tree(torch.full((B,), -1, dtype=torch.int32, device="cuda"), [1] * B, B, 1)

    def forward(tokens, t, pools, lens, seq):
        rows = k4.linear_w4(embed[tokens], qkv).view(-1, 3 * H, D)
        q, k = k4.qk_norm_rotary(rows[:, :H], rows[:, H:2 * H], B, None, rotary, positions=lens.lens[seq] + t.depths)
        v = rows[:, 2 * H:]
        ctx = k4.decode_attn_tree(q, k, v, *pools, lens, table, t)
        logits = k4.linear_w4(embed[tokens] + ctx.view(-1, hid), head)
        path, taken, following = k4.accept_drafts(logits, tokens, t)
        k4.kv_pages_extend(k, v, *pools, lens, table, t, path, taken)
        lens.lens.add_(taken)
        return path, taken, following

    def lengths():
        lens = torch.tensor(start, dtype=torch.int32, device="cuda")
        return SeqInfo(lens, None, B, None, lens)
    # one token a step
    pools1, lens1, newest = [p.clone() for p in context], lengths(), torch.tensor([3, 4, 5], device="cuda")
    greedy, seq1 = [newest], torch.arange(B, device="cuda")
    for _ in range(steps * 8):
        newest = forward(newest, one, pools1, lens1, seq1)[2]
        greedy.append(newest)
    greedy = torch.stack(greedy, 1).tolist()
    # drafted trees, whose nodes are partly right
    pools, lens = [p.clone() for p in context], lengths()
    seq = torch.repeat_interleave(torch.arange(B, device="cuda"), torch.tensor(counts, device="cuda"))
    tokens = torch.zeros(T, dtype=torch.int64, device="cuda")
    taken = [0] * B
    captured = None
    if graph:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        scratch = [p.clone() for p in context]
        with torch.cuda.stream(side):
            warm = lengths()
            forward(tokens, tree, scratch, warm, seq)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured):
            result = forward(tokens, tree, pools, lens, seq)
    announce("steps together", graph)
    for i in range(steps):
        left = [row[n:] for row, n in zip(greedy, taken)]
        tokens.copy_(torch.tensor(_drafted(left, counts, parents, V, i)))
        if graph:
            captured.replay()
        else:
            result = forward(tokens, tree, pools, lens, seq)
        want = []
        first = 0
        for b, n in enumerate(counts):
            cur, way = 0, [0]
            while True:
                fits = [c for c in range(n) if parents[first + c] == cur and int(tokens[first + c]) == left[b][len(way)]]
                if not fits:
                    break
                cur = fits[0]
                way.append(cur)
            want.append(way)
            first += n
        assert [row[:n] for row, n in zip(result[0].tolist(), result[1].tolist())] == want, i
        taken = [n + len(w) for n, w in zip(taken, want)]
        assert result[2].tolist() == [row[n] for row, n in zip(greedy, taken)]
    assert sum(taken) > steps * B                        # some drafts were accepted
    assert lens.lens.tolist() == [n + m for n, m in zip(start, taken)]
    for b in range(B):
        for p, p1 in zip(pools, pools1):
            rows, rows1 = (x[table[b].long()].transpose(0, 1).reshape(H, -1, D)[:, :start[b] + taken[b]].float() for x in (p, p1))
            # of the same numbers, by products that may add them up in another order
            assert ((rows - rows1).abs() <= 2 ** -9 * (rows1.abs() + 1)).all()
