"""Caches in 8 bits that are views: dimensions of one have no stride that matters, whatever it is."""
import pytest
import torch

from gpu_util import announce
from test_gpu_kv8 import rows_of

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
I8, E4 = torch.int8, torch.float8_e4m3fn


def _odd(t, dim):
    """The same elements, with the stride of a dimension of one set to an odd number."""
    assert t.shape[dim] == 1
    strides = list(t.stride())
    strides[dim] = 7
    return t.as_strided(t.shape, strides, t.storage_offset())


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("N,H,P,odd", [
    (5, 1, 32, [(0, 1), (1, 1), (2, 1), (3, 1)]),                 # one head
    (1, 3, 64, [(0, 0), (1, 0), (2, 0), (3, 0)]),                 # one page
    (5, 2, 16, [(1, 2), (2, 2), (3, 2)]),                         # one block a page
    (1, 1, 16, [(0, 0), (0, 1), (1, 0), (1, 1), (1, 2), (2, 0), (2, 1), (2, 2), (3, 0)]),
])
def test_dimensions_of_one(native, N, H, P, odd):
    import energonai_amd.kernel as K
    from energonai_amd.seqinfo import build_seq_info
    announce("kv8 dimensions of one", native, N, H, P)
    D, dtype, code = 64, BF16, E4
    g = torch.Generator().manual_seed(N + H)
    n = min(N * P, 48)                                            # the appended position completes a block
    ks, vs = rows_of(1, H, D, [n], dtype, g), rows_of(1, H, D, [n], dtype, g)
    k, v = ks[0].transpose(0, 1).cuda(), vs[0].transpose(0, 1).cuda()
    q = torch.randn(1, 2 * H, 1, D, generator=g).to(dtype).cuda()

    def run(change):
        cache = list(K.kv8_pages(N, 1, H, P, D, -(-n // P), dtype, "cuda", code))
        cache[6].copy_(torch.arange(cache[6].shape[1]).flip(0)[None])
        for i, dim in change:
            cache[i] = _odd(cache[i], dim)
        lens = torch.tensor([n - 1], dtype=torch.int32).cuda()
        info, now = build_seq_info(lens, 1), build_seq_info(lens + 1, 1)
        if not native:                                            # the general call
            info, now = lens, lens + 1
        K.kv8_pages_fill(k[:n - 1], v[:n - 1], cache, 1, n - 1, info)
        turned = K.kv8_pages_append(q[:, :, 0], k[n - 1:], v[n - 1:], cache, info)
        return (turned,) + K.kv8_pages_read(cache, now, n) + (K.decode_attn_kv8(q, cache, now),)
    for a, b in zip(run([]), run(odd)):
        assert torch.equal(a, b)


def test_results_over_one_another():
    """Two results of one read, or a context that lies partly over the queries, are refused; over the queries as a whole it may lie."""
    import energonai_amd.kernel as K
    announce("kv8 results over one another")
    B, H, D, P = 3, 2, 64, 16
    cache = K.kv8_pages(3, B, H, P, D, 1, F16, "cuda")
    cache.page_table.copy_(torch.arange(3)[:, None])
    x = torch.randn(27, 2 * H, D, device="cuda").half()
    lens = torch.tensor([9, 9, 9], dtype=torch.int32).cuda()
    K.kv8_pages_fill(x[:, :H], x[:, H:], cache, B, 9, lens)
    k, v = K.kv8_pages_read(cache, lens, 12)
    two = torch.empty(2, B, H, 12, D, device="cuda", dtype=F16)
    got = K.kv8_pages_read(cache, lens, 12, out=(two[0], two[1]))
    assert torch.equal(got[0], k) and torch.equal(got[1], v)
    flat = torch.empty(two[0].numel() + 8, device="cuda", dtype=F16)
    over = flat[:-8].view(k.shape), flat[8:].view(k.shape)
    for out in ((two[0], two[0]), over, (over[1], over[0]), (two[0],), (two[0], two[1], two[1])):
        with pytest.raises(RuntimeError):
            K.kv8_pages_read(cache, lens, 12, out=out)
    q = torch.randn(B, 4, 1, D, device="cuda").half()
    want = K.decode_attn_kv8(q, cache, lens)
    flat = torch.zeros(q.numel() + 64, device="cuda", dtype=F16)
    qv = flat[:-64].view(q.shape)
    qv.copy_(q)
    with pytest.raises(RuntimeError):
        K.decode_attn_kv8(qv, cache, lens, out=flat[64:].view(q.shape))
    assert K.decode_attn_kv8(qv, cache, lens, out=qv) is qv and torch.equal(qv, want)
