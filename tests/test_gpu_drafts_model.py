"""Steps of drafted nodes and weights in 4 bits through the model layers."""
import copy

import pytest
import torch

from gpu_util import announce

pytestmark = pytest.mark.gpu

HID, HEADS = 256, 4


def _block(dtype, **kw):
    from energonai_amd.model import Block1D
    torch.manual_seed(3)
    return Block1D(HID, HEADS, 2, activation=kw.pop("activation", torch.nn.functional.relu), dtype=dtype, max_seq_len=128, kv_page_size=16, **kw).cuda().eval()


def _prompt(lens, dtype, seed=1):
    g = torch.Generator().manual_seed(seed)
    x = torch.zeros(len(lens), max(lens), HID, dtype=dtype)
    for b, n in enumerate(lens):
        x[b, max(lens) - n:] = torch.randn(n, HID, generator=g).to(dtype)
    return x.cuda()


@pytest.mark.parametrize("turn", [{}, dict(rotary_dim=32, qk_norm=True)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@torch.no_grad()
def test_nodes_are_the_steps_they_stand_for(dtype, turn):
    """A chain of nodes gives what steps of one token give; so does each way of a tree; and the accepted rows continue the cache."""
    from energonai_amd import kernel as K
    from energonai_amd.model import PackedStack
    lens, B = [17, 30, 5], 3
    blocks = [_block(dtype, **turn) for _ in range(2)]
    stack, other = PackedStack(blocks), PackedStack([copy.deepcopy(b) for b in blocks])
    x, lens_d = _prompt(lens, dtype), torch.tensor(lens, dtype=torch.int32, device="cuda")
    for s in (stack, other):
        s(x, first_cache=True, seq_lens=lens_d)
    g = torch.Generator(device="cuda").manual_seed(5)
    parents = [-1, 0, 1, 1] * B                              # two ways: 0 1 2 and 0 1 3
    rows = torch.randn(B, 4, HID, generator=g, device="cuda", dtype=dtype)
    tree = K.draft_tree(torch.tensor(parents, dtype=torch.int32, device="cuda"), [4] * B, B, 4)
    announce("nodes of a stack", dtype, turn)
    got = stack.forward_nodes(rows.view(1, -1, HID), tree).view(B, 4, HID)
    want = [other(rows[:, i:i + 1], first_cache=False)[:, -1] for i in (0, 1, 3)]
    # both round activations to 16 bits, in other orders of the same sums, through two blocks: a few steps of each
    tol = 2 ** -8 if dtype == torch.float16 else 2 ** -5
    for i, w in zip((0, 1, 3), want):
        assert ((got[:, i] - w).abs() <= tol * (1 + w.abs())).all(), i
    path = torch.tensor([[0, 1, 3, -1]] * B, dtype=torch.int32, device="cuda")
    stack.accept_nodes(path, torch.full((B,), 3, dtype=torch.int32, device="cuda"))
    for a, b in zip(stack.blocks, other.blocks):
        assert a.attn.kv_cache.lens.tolist() == b.attn.kv_cache.lens.tolist() == [n + 3 for n in lens]
        assert a.attn.kv_cache._host_lens == b.attn.kv_cache._host_lens
    after = torch.randn(B, 1, HID, generator=g, device="cuda", dtype=dtype)
    one = K.draft_tree(torch.full((B,), -1, dtype=torch.int32, device="cuda"), [1] * B, B, 1)
    got, w = stack.forward_nodes(after.view(1, B, HID), one).view(B, HID), other(after, first_cache=False)[:, -1]
    assert ((got - w).abs() <= tol * (1 + w.abs())).all()
    # sequences of different counts, one of them with nothing
    stack.accept_nodes(torch.zeros(B, 1, dtype=torch.int32, device="cuda"), torch.tensor([1, 0, 1], dtype=torch.int32, device="cuda"))
    assert stack.blocks[0].attn.kv_cache.lens.tolist() == [n + 3 + m for n, m in zip(lens, (1, 0, 1))]


@torch.no_grad()
def test_refusals():
    from energonai_amd import kernel as K
    from energonai_amd.model import Block1D, PagedKVCache8
    tree = K.draft_tree(torch.full((1,), -1, dtype=torch.int32, device="cuda"), [1], 1, 1)
    x = torch.zeros(1, 1, HID, dtype=torch.float16, device="cuda")
    b = _block(torch.float16)
    with pytest.raises(RuntimeError, match="first_cache"):
        b.forward_nodes(x, tree)
    b(_prompt([5], torch.float16), first_cache=True)
    with pytest.raises(RuntimeError, match="forward_nodes"):
        b.accept_nodes(torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda"))
    whole = Block1D(HID, HEADS, 2, dtype=torch.float16, max_seq_len=64).cuda()
    whole(_prompt([5], torch.float16), first_cache=True)
    with pytest.raises(RuntimeError, match="kv_page_size"):
        whole.forward_nodes(x, tree)
    eight = Block1D(HID, HEADS, 2, dtype=torch.float16, max_seq_len=64, kv_cache_dtype=torch.int8).cuda()
    eight(_prompt([5], torch.float16), first_cache=True)
    assert type(eight.attn.kv_cache) is PagedKVCache8
    with pytest.raises(RuntimeError, match="16-bit"):
        eight.forward_nodes(x, tree)
    # a pool that is used up keeps its lengths
    b.forward_nodes(x, tree)
    cache = b.attn.kv_cache
    cache._free.clear()
    cache._host_lens = [16]
    with pytest.raises(RuntimeError, match="used up"):
        b.accept_nodes(torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda"))
    assert cache.lens.tolist() == [5]


@torch.no_grad()
def test_nodes_of_a_cache_that_has_gone_on_are_refused():
    """Once the cache has taken in anything else, the rows of an earlier step of nodes do not belong behind it."""
    from energonai_amd import kernel as K
    tree = K.draft_tree(torch.tensor([-1, 0], dtype=torch.int32, device="cuda"), [2], 1, 2)
    x, one = torch.randn(1, 2, HID, dtype=torch.float16, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    path = torch.tensor([[0, -1]], dtype=torch.int32, device="cuda")
    announce("nodes of a cache that has gone on")
    b = _block(torch.float16)
    for between in (lambda: b(x[:, :1], first_cache=False), lambda: b(_prompt([9], torch.float16), first_cache=True),
                    lambda: b.attn.kv_cache.extend(*b.attn._nodes[:3], path, one)):
        b(_prompt([5], torch.float16), first_cache=True)
        b.forward_nodes(x, tree)
        between()
        lens = b.attn.kv_cache.lens.tolist()
        with pytest.raises(RuntimeError, match="gone on"):
            b.accept_nodes(path, one)
        assert b.attn.kv_cache.lens.tolist() == lens
        with pytest.raises(RuntimeError, match="forward_nodes"):
            b.accept_nodes(path, one)
    # the nodes may be gone over again, and finished sequences released
    b.forward_nodes(x, tree)
    b.forward_nodes(x, tree)
    b.attn.kv_cache.release(0)
    b.accept_nodes(path, torch.zeros_like(one))
    assert b.attn.kv_cache.lens.tolist() == [0]


@torch.no_grad()
def test_rotated_nodes_whose_counts_say_more_than_there_is():
    """Offsets past the rows of a call: every row of it has its own sequence's position, and nothing past them is written."""
    from energonai_amd import kernel as K
    from energonai_amd.seqinfo import build_seq_info
    b = _block(torch.float16, rotary_dim=32)
    b(_prompt([5, 9], torch.float16), first_cache=True, seq_lens=torch.tensor([5, 9], dtype=torch.int32, device="cuda"))
    x = torch.randn(1, 3, HID, dtype=torch.float16, device="cuda")
    parents = torch.tensor([-1, 0, -1], dtype=torch.int32, device="cuda")
    announce("counts past the rows")
    got = b.forward_nodes(x, K.draft_tree(parents, build_seq_info([2, 60], 2), 2, 64))
    want = b.forward_nodes(x, K.draft_tree(parents, [2, 1], 2, 64))
    assert torch.equal(got, want)


@pytest.mark.parametrize("activation", [torch.nn.functional.relu, torch.nn.GELU(), torch.nn.GELU(approximate="tanh"), torch.nn.functional.silu])
@pytest.mark.parametrize("zero_points", [False, True])
@torch.no_grad()
def test_block_with_weights_in_4_bits(activation, zero_points):
    """A block whose projections are replaced gives, for prompts and steps, what a block gives whose weights are the rounded ones."""
    from energonai_amd.model import Linear4, quantize_linears
    dtype, lens = torch.float16, [9, 33]
    plain = _block(dtype, activation=activation)
    small = quantize_linears(copy.deepcopy(plain), 64, zero_points)
    layers = [(n, m) for n, m in small.named_modules() if isinstance(m, Linear4)]
    assert sorted(n for n, _ in layers) == ["attn.dense", "attn.query_key_value", "mlp.dense_1", "mlp.dense_2"]
    announce("4-bit block", activation, zero_points)
    for n, m in layers:
        eye = torch.eye(m.in_features, dtype=dtype, device="cuda")
        bias = m.bias
        m.bias = None
        plain.get_submodule(n).weight.copy_(m(eye).t())       # rounded to 16 bits
        m.bias = bias
    x, lens_d = _prompt(lens, dtype), torch.tensor(lens, dtype=torch.int32, device="cuda")
    step = torch.randn(2, 1, HID, device="cuda", dtype=dtype)
    for got, want in ((small(x, first_cache=True, seq_lens=lens_d), plain(x, first_cache=True, seq_lens=lens_d)), (small(step), plain(step))):
        # both round activations and (the plain one) weights to fp16, in other orders of the same sums
        assert ((got - want).abs() <= 2 ** -7 * (1 + want.abs())).all()
    state = small.state_dict()
    again = quantize_linears(copy.deepcopy(plain), 64, zero_points)
    again.load_state_dict(state)
    assert torch.equal(again(x, first_cache=True, seq_lens=lens_d), small(x, first_cache=True, seq_lens=lens_d))


@torch.no_grad()
def test_padding_rows_of_rotated_nodes_do_not_change_from_call_to_call():
    """Rows behind the last sequence are rotated by that sequence's length, not by what memory held."""
    from energonai_amd import kernel as K
    b = _block(torch.float16, rotary_dim=32)
    b(_prompt([5, 9], torch.float16), first_cache=True, seq_lens=torch.tensor([5, 9], dtype=torch.int32, device="cuda"))
    x = torch.randn(1, 40, HID, dtype=torch.float16, device="cuda")
    parents = torch.full((40,), -1, dtype=torch.int32, device="cuda")
    announce("padding rows of rotated nodes")
    first = None
    for fill in (0, 1 << 20, -5):
        poison = [torch.full((40,), fill, dtype=t, device="cuda") for t in (torch.int64, torch.int32) for _ in range(8)]
        torch.cuda.synchronize()
        del poison
        b.forward_nodes(x, K.draft_tree(parents, [2, 1], 2, 2))
        keys = b.attn._nodes[0].clone()
        first = keys if first is None else first
        assert torch.equal(keys, first)


@torch.no_grad()
def test_released_sequences_accept_nothing():
    """A sequence that was released after its nodes were gone over has no place for them; the others' nodes, and none of its own, may be accepted still."""
    from energonai_amd import kernel as K
    b = _block(torch.float16)
    lens = torch.tensor([5, 9], dtype=torch.int32, device="cuda")
    tree = K.draft_tree(torch.tensor([-1, 0] * 2, dtype=torch.int32, device="cuda"), [2, 2], 2, 2)
    x = torch.randn(1, 4, HID, dtype=torch.float16, device="cuda")
    path = torch.tensor([[0, 1], [0, 1]], dtype=torch.int32, device="cuda")
    announce("released sequences")
    for host in (False, True):
        b(_prompt([5, 9], torch.float16), first_cache=True, seq_lens=lens)
        b.forward_nodes(x, tree)
        cache = b.attn.kv_cache
        cache.release(0)
        both = torch.tensor([2, 2], dtype=torch.int32, device="cuda")
        with pytest.raises(RuntimeError, match="released"):
            b.accept_nodes(path, both, [2, 2] if host else None)
        assert cache.lens.tolist() == [0, 9] and cache._host_lens == [0, 9] and cache.pages_in_use() == 1
        b.accept_nodes(path, torch.tensor([0, 2], dtype=torch.int32, device="cuda"), [0, 2] if host else None)
        assert cache.lens.tolist() == [0, 11] and cache._host_lens == [0, 11]


@torch.no_grad()
def test_stacks_accept_in_all_blocks_or_in_none():
    """One block whose cache has no place for the nodes keeps them out of the others' too."""
    from energonai_amd import kernel as K
    from energonai_amd.model import PackedStack
    stack = PackedStack([_block(torch.float16) for _ in range(2)])
    tree = K.draft_tree(torch.tensor([-1, 0], dtype=torch.int32, device="cuda"), [2], 1, 2)
    x, one = torch.randn(1, 2, HID, dtype=torch.float16, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    path = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    announce("stacks accept in all blocks or in none")
    stack(_prompt([5], torch.float16), first_cache=True)
    stack.forward_nodes(x, tree)
    stack.blocks[1].attn.kv_cache.release(0)
    with pytest.raises(RuntimeError, match="released"):
        stack.accept_nodes(path, one)
    assert stack.blocks[0].attn.kv_cache.lens.tolist() == [5]
    stack(_prompt([5], torch.float16), first_cache=True)
    stack.forward_nodes(x, tree)
    stack.accept_nodes(path, one)
    assert [b.attn.kv_cache.lens.tolist() for b in stack.blocks] == [[6], [6]]


@pytest.mark.parametrize("turn", [{}, dict(rotary_dim=32)])
@torch.no_grad()
def test_nodes_do_not_keep_what_they_belong_to(turn):
    """A step of nodes that is never accepted holds no cache that was replaced or taken away, and no rows once the cache has gone on."""
    import gc
    import weakref

    from energonai_amd import kernel as K
    b = _block(torch.float16, **turn)
    tree = K.draft_tree(torch.tensor([-1, 0], dtype=torch.int32, device="cuda"), [2], 1, 2)
    x, one = torch.randn(1, 2, HID, dtype=torch.float16, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    path = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    announce("nodes that are not accepted", turn)

    def gone():
        gc.collect()
        return cache() is None
    for between, takes_cache in ((lambda: b(_prompt([9], torch.float16), first_cache=True), True), (lambda: b(x[:, :1], first_cache=False), False),
                                 (lambda: setattr(b.attn, "kv_cache", None), True)):
        b(_prompt([5], torch.float16), first_cache=True)
        b.forward_nodes(x, tree)
        cache, rows = weakref.ref(b.attn.kv_cache), weakref.ref(b.attn._nodes[0])
        between()
        assert gone() == takes_cache
        assert not takes_cache or b.attn.kv_cache is None or rows() is None
        if not takes_cache:
            assert rows() is None
        with pytest.raises(RuntimeError, match="gone on"):
            b.accept_nodes(path, one)
        assert rows() is None


@torch.no_grad()
def test_layers_of_several_names_are_one_layer():
    """A layer that is there twice is replaced at both places by one; a layer that cannot be replaced leaves all as they were."""
    from energonai_amd.model import Linear4, quantize_linears
    shared = torch.nn.Linear(64, 32, dtype=torch.float16, device="cuda")
    m = torch.nn.Module()
    m.a, m.b, m.inner = shared, shared, torch.nn.Sequential(shared, torch.nn.ReLU())
    announce("layers of several names")
    quantize_linears(m, 32)
    assert type(m.a) is Linear4 and m.a is m.b is m.inner[0]
    bad = torch.nn.Sequential(torch.nn.Linear(64, 32, dtype=torch.float16, device="cuda"), torch.nn.Linear(32, 8, dtype=torch.float32, device="cuda"))
    with pytest.raises(RuntimeError):
        quantize_linears(bad, 32)
    assert all(type(layer) is torch.nn.Linear for layer in bad)
    # a layer's 16-bit weight goes before the next is turned: the most that many layers take is what one takes
    most = []
    for n in (1, 24):
        many = torch.nn.Sequential(*[torch.nn.Linear(2048, 2048, dtype=torch.float16, device="cuda") for _ in range(n)])
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        quantize_linears(many, 128)
        most.append(torch.cuda.max_memory_allocated() - before)
        assert torch.cuda.memory_allocated() < before
    assert most[1] <= most[0]


@torch.no_grad()
def test_counts_past_the_path_are_refused():
    """Lengths do not go on past the rows that a path has: the positions behind them would hold what the pages held."""
    from energonai_amd import kernel as K
    b = _block(torch.float16)
    b(_prompt([5, 9], torch.float16), first_cache=True, seq_lens=torch.tensor([5, 9], dtype=torch.int32, device="cuda"))
    tree = K.draft_tree(torch.tensor([-1, 0] * 2, dtype=torch.int32, device="cuda"), [2, 2], 2, 2)
    announce("counts past the path")
    b.forward_nodes(torch.randn(1, 4, HID, dtype=torch.float16, device="cuda"), tree)
    path = torch.tensor([[0, 1], [0, 1]], dtype=torch.int32, device="cuda")
    cache, pages = b.attn.kv_cache, b.attn.kv_cache.pages_in_use()
    for counts in ([3, 1], [1, -1], [1]):
        with pytest.raises(RuntimeError, match="counts"):
            b.accept_nodes(path, torch.tensor(counts, dtype=torch.int32, device="cuda"))
    assert cache.lens.tolist() == [5, 9] and cache._host_lens == [5, 9] and cache.pages_in_use() == pages
    b.accept_nodes(path, torch.tensor([2, 1], dtype=torch.int32, device="cuda"))
    assert cache.lens.tolist() == [7, 10]


@torch.no_grad()
def test_single_steps_after_accepted_nodes():
    """An ordinary step goes on behind the accepted nodes: its newest position is the one that single steps give.  The positions before it are those of
    the calls that return them: accepted nodes are not among them."""
    from energonai_amd import kernel as K
    lens, B, dtype = [17, 5], 2, torch.float16
    b = _block(dtype)
    other = copy.deepcopy(b)
    g = torch.Generator(device="cuda").manual_seed(15)
    rows, after = (torch.randn(B, n, HID, generator=g, device="cuda", dtype=dtype) for n in (2, 1))
    lens_d = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for m in (b, other):
        m(_prompt(lens, dtype), first_cache=True, seq_lens=lens_d)
    tree = K.draft_tree(torch.tensor([-1, 0] * B, dtype=torch.int32, device="cuda"), [2] * B, B, 2)
    announce("single steps after accepted nodes")
    b.forward_nodes(rows.view(1, -1, HID), tree)
    b.accept_nodes(torch.tensor([[0, 1]] * B, dtype=torch.int32, device="cuda"), torch.full((B,), 2, dtype=torch.int32, device="cuda"))
    for i in range(2):
        other(rows[:, i:i + 1], first_cache=False)
    got, want = b(after, first_cache=False), other(after, first_cache=False)
    # both round activations to 16 bits, in other orders of the same sums: a few steps of each
    assert ((got[:, -1] - want[:, -1]).abs() <= 2 ** -8 * (1 + want[:, -1].abs())).all()
    assert got.shape[1] == max(lens) + 1 and want.shape[1] == max(lens) + 3
    assert b.attn.kv_cache.lens.tolist() == other.attn.kv_cache.lens.tolist() == [n + 3 for n in lens]
