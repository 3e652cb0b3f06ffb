"""Steps of drafted tokens at their edges: rows that are no node's, nodes that no call of the tree has, weights far below the largest."""
import math

import pytest
import torch

from gpu_util import announce

pytestmark = pytest.mark.gpu


def K():
    from energonai_amd import kernel
    return kernel


@pytest.mark.parametrize("counts,rows", [([3, 0, 2], 5 + 70), ([3, 0, 2], 6), ([0, 0], 4), ([64, 70], 64 + 70 + 200), ([2, 60], 3), ([5], 5)])
def test_rows_behind_the_last_sequence_have_no_node(counts, rows):
    """Masks and depths of rows that no sequence has are zeros, whatever was in the memory; nothing past the rows is written."""
    from energonai_amd import _lib
    from energonai_amd.seqinfo import build_seq_info
    info = build_seq_info(counts, len(counts))
    parents = torch.arange(rows, dtype=torch.int32, device="cuda") % 3 - 1
    masks = torch.full((rows + 8,), -7, dtype=torch.int64, device="cuda")
    depths = torch.full((rows + 8,), 99, dtype=torch.int32, device="cuda")
    announce("rows behind the last sequence", counts, rows)
    status = _lib.fn.en_draft_tree(parents.data_ptr(), info.cu_seqlens.data_ptr(), len(counts), rows, masks.data_ptr(), depths.data_ptr(), _lib.stream_of(parents))
    assert status == 0
    there = min(sum(counts), rows)
    assert (masks[there:rows] == 0).all() and (depths[there:rows] == 0).all()
    assert (masks[rows:] == -7).all() and (depths[rows:] == 99).all()
    nodes, at = [], 0
    for n in counts:
        nodes += [at + i for i in range(min(n, 64)) if at + i < rows]
        at += n
    assert (masks[nodes] != 0).all() and (depths[nodes] < 64).all()


def test_extension_knows_the_largest_number_of_nodes():
    """Entries of a path that name nodes past the tree's ``max_nodes`` are passed over, by the native call and by the checked one."""
    from energonai_amd.seqinfo import build_seq_info
    counts, H, D, P, dtype = [6, 3], 2, 64, 16, torch.float16
    g = torch.Generator().manual_seed(5)
    k, v = (torch.randn(9, H, D, generator=g).to(dtype).cuda() for _ in range(2))
    lens = torch.tensor([3, 20], dtype=torch.int32, device="cuda")
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device="cuda")
    tree = K().draft_tree(torch.full((9,), -1, dtype=torch.int32, device="cuda"), counts, 2, 4)
    path = torch.tensor([[0, 3, 4, 5], [2, 1, 3, 0]], dtype=torch.int32, device="cuda")
    taken = torch.full((2,), 4, dtype=torch.int32, device="cuda")
    announce("extension and the largest number of nodes")
    for at in (build_seq_info([3, 20], 2), lens):
        pools = [torch.zeros(4, H, P, D, dtype=dtype, device="cuda") for _ in range(2)]
        lost = torch.zeros(1, dtype=torch.int32, device="cuda")
        K().kv_pages_extend(k, v, *pools, at, table, tree, path, taken, overflow=lost)
        for pool, new in zip(pools, (k, v)):
            want = torch.zeros_like(pool)
            want[0, :, 3], want[0, :, 4] = new[0], new[3]                      # nodes 4 and 5 are past the largest
            want[3, :, 4], want[3, :, 5], want[3, :, 7] = new[8], new[7], new[6]    # ... and 3 is none of the sequence's
            assert torch.equal(pool, want)
        assert int(lost) == 0


@pytest.mark.parametrize("G", [4, 12, 32])
def test_weights_far_below_the_largest(G):
    """fp16: one position whose weight is 2^27 times that of each of 60000 others.  Together they are 4.5e-4 of the result.

    Weights are kept down to 2^-32 of the largest, so each of n others is off by at most that much of it; beside it, half a step of the result, and in
    the fp32 sums n additions of 2^-24 each of what they add up to."""
    B, H, D, P, n, dtype = 64, 8, 64, 64, 60000, torch.float16
    pages = -(-n // P)
    kp, vp = torch.zeros(pages, H, P, D, dtype=dtype, device="cuda"), torch.ones(pages, H, P, D, dtype=dtype, device="cuda")
    kp[0, :, 5, 0] = 18.71875
    vp[0, :, 5] = 0
    table = torch.arange(pages, dtype=torch.int32, device="cuda").repeat(B, 1)             # all sequences read the same pages: a workgroup has a whole one
    nodes = 8
    q = torch.zeros(B * nodes, H * G, D, dtype=dtype, device="cuda")
    q[:, :, 0] = 1
    new_k, new_v = torch.zeros(B * nodes, H, D, dtype=dtype, device="cuda"), torch.ones(B * nodes, H, D, dtype=dtype, device="cuda")
    tree = K().draft_tree(torch.full((B * nodes,), -1, dtype=torch.int32, device="cuda"), [nodes] * B, B, nodes)
    announce("weights far below the largest", G)
    got = K().decode_attn_tree(q, new_k, new_v, kp, vp, torch.full((B,), n, dtype=torch.int32, device="cuda"), table, tree, scale=1.0).double()
    w = n * math.exp(-18.71875)                              # n - 1 positions and the node itself
    want = w / (1 + w)
    tolerance = n * 2.0 ** -32 + 2.0 ** -11 * want + 2 * n * 2.0 ** -24 * want
    assert tolerance < want / 8
    assert float((got - want).abs().max()) <= tolerance, (float(got.min()), float(got.max()), want)
