"""Tree attention whose tiles are shared out over workgroups in runs of several: parts of units at either end of a run, whole ones between."""
import random

import pytest
import torch

from gpu_util import announce
from oracle import drafts as ref
from test_gpu_drafts import tolerance, trees

pytestmark = pytest.mark.gpu


def K():
    from energonai_amd import kernel
    return kernel


def shares(lens, counts, G, H, most, tile, at_once, groups):
    """Of the runs that the workgroups have: how many units' parts begin inside a run (and so are a run's second part), how many runs hold the
    end of one unit, whole ones and the beginning of another, and the tiles of a run.  A unit counts one more tile for its end."""
    units = [-(-(n + m) // tile) for n, m in zip(lens, counts) if m for _ in range(H * -(-min(m, most) * G // at_once))]
    total = sum(u + 1 for u in units)
    quota = -(-total // groups)
    second, both, x = 0, 0, 0
    kinds = {}
    for u in units:
        w0, w1 = x // quota, (x + u - 1) // quota
        if w0 == w1:
            kinds.setdefault(w0, []).append("whole")
        else:
            if x - w0 * quota > 1:
                second += 1
            kinds.setdefault(w0, []).append("head")
            for w in range(w0 + 1, w1):
                kinds.setdefault(w, []).append("middle")
            kinds.setdefault(w1, []).append("tail")
        x += u + 1
    both = sum(1 for k in kinds.values() if k[0] == "tail" and k[-1] == "head" and "whole" in k)
    return second, both, quota


def reference(q, k_new, v_new, k_pool, v_pool, lens, table, masks, counts):
    """As ``oracle.drafts.attend``, a head at a time."""
    T, Hq, D = q.shape
    H, G = k_pool.shape[1], Hq // k_pool.shape[1]
    out, size, most, first = torch.zeros(T, Hq, D, dtype=torch.float64), torch.zeros(T, Hq, D, dtype=torch.float64), torch.zeros(T, Hq, 1, dtype=torch.float64), 0
    for b, (n, m) in enumerate(zip(lens, counts)):
        if m == 0:
            continue
        ids = table[b, :-(-n // k_pool.shape[2])].long()
        rows = slice(first, first + m)
        seen = torch.tensor([[w >> i & 1 for i in range(m)] for w in masks[first:first + m]], dtype=torch.bool)
        for h in range(H):
            k, v = (torch.cat((pool[ids, h].reshape(-1, D)[:n], new[rows, h])).double() for pool, new in ((k_pool, k_new), (v_pool, v_new)))
            x = q[rows, h * G:(h + 1) * G].double().reshape(m * G, D)
            s = x @ k.t() * D ** -0.5
            visible = torch.cat((torch.ones(m, n, dtype=torch.bool), seen), 1).repeat_interleave(G, 0)
            p = torch.softmax(s.masked_fill(~visible, float("-inf")), 1)
            out[rows, h * G:(h + 1) * G], size[rows, h * G:(h + 1) * G] = (p @ v).view(m, G, D), (p @ v.abs()).view(m, G, D)
            most[rows, h * G:(h + 1) * G] = (x.abs() @ k.abs().t() * D ** -0.5).masked_fill(~visible, 0).amax(1).view(m, G, 1)
        first += m
    return out, size, most


CASES = [
    # rows at a time, query heads a key head, nodes, sequences, key heads, head size, workgroups
    (16, 2, 8, 100, 8, 64, 512),
    (16, 1, 3, 110, 8, 128, 512),
    (64, 4, 12, 70, 8, 64, 512),
    (128, 5, 20, 70, 8, 64, 512),
    (128, 2, 64, 120, 4, 96, 512),
    (256, 4, 50, 24, 8, 64, 256),
    (256, 8, 63, 40, 4, 128, 256),          # two runs of rows a unit
]


def sizes(at_once, G, nodes, B):
    """Long and short caches in turn, sequences without either among them."""
    r = random.Random(at_once + G)
    lens = [2000, 0, 1, 127, 128] + [r.randrange(1, 2000) if b % 2 else r.choice([0, 30, 100, 129, 260]) for b in range(B - 5)]
    counts = [nodes, 1, nodes, 0, nodes] + [r.choice([0, 1, nodes, r.randint(1, nodes)]) for _ in range(B - 5)]
    return lens, counts


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("at_once,G,nodes,B,H,D,groups", CASES)
def test_runs_of_several_tiles(at_once, G, nodes, B, H, D, groups, dtype):
    P, longest = 64, 2000
    lens, counts = sizes(at_once, G, nodes, B)
    assert at_once == next(n for n in (16, 64, 128, 256) if nodes * G <= n or n == 256)
    second, both, quota = shares(lens, counts, G, H, nodes, 128 if at_once == 16 else 64, at_once, groups)
    assert quota >= 3 and second >= 20 and both >= 1
    g = torch.Generator().manual_seed(at_once * 8 + G)
    held = [-(-n // P) for n in lens]
    N = sum(held) + 3
    ids, table, at = torch.randperm(N, generator=g, dtype=torch.int32), torch.full((B, longest // P + 2), -1, dtype=torch.int32), 0
    for b, n in enumerate(held):
        table[b, :n] = ids[at:at + n]
        at += n
    pools = [torch.randn(N, H, P, D, generator=g).to(dtype) for _ in range(2)]
    T = sum(counts)
    q, k, v = (torch.randn(T, h, D, generator=g).to(dtype) for h in (G * H, H, H))
    need = K().decode_attn_tree_workspace_bytes(B, G * H, H, table.shape[1] * P, D, nodes)
    assert need == 2 * groups * at_once * (4 * D + 8) + 4 * (B + 1)         # shared out, and so many rows at a time over so many workgroups
    parents = trees(counts, G)
    tree = K().draft_tree(torch.tensor(parents, dtype=torch.int32, device="cuda"), counts, B, nodes)
    masks, _ = ref.masks(parents, counts)
    want, size, most = reference(q, k, v, *pools, lens, table, masks, counts)
    announce("runs of several tiles", at_once, G, nodes, B, H, D, dtype, "quota", quota, "second parts", second, "of both", both)
    dev = [t.cuda() for t in (q, k, v, *pools, torch.tensor(lens, dtype=torch.int32), table)]
    # what the buffer holds before is of no consequence, and neither is what a run before left there
    workspace = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    for _ in range(2):
        got = K().decode_attn_tree(*dev, tree, workspace=workspace).cpu()
        off = (got.double() - want).abs() - tolerance(want, size, most, dtype, D, longest + 64)
        assert float(off.max()) <= 0, float(off.max())
    assert torch.equal(K().decode_attn_tree(*dev, tree).cpu(), got)
