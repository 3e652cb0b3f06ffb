"""Steps of drafted tokens at their edges: rows that are no node's, nodes that no call of the tree has, weights far below the largest."""
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
