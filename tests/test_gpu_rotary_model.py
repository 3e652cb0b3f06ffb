"""Blocks with rotary positions and norms of heads, on every kind of cache, and the operators behind them run together as they would be used."""
import pytest
import torch

from gpu_util import announce, max_abs
from oracle import kv8 as ref

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _mods():
    import energonai_amd.kernel as K
    import energonai_amd.model as M
    return K, M


def _seed(module, g):
    with torch.no_grad():
        for name, prm in module.named_parameters():
            if prm.dim() > 1:
                prm.copy_(torch.randn(prm.shape, generator=g) / prm.shape[1] ** 0.5)
            else:
                prm.copy_((1.0 if name.endswith("weight") or "norm" in name else 0.0) + 0.05 * torch.randn(prm.shape, generator=g))


def _layer_norm(x, w, b, eps):
    return torch.nn.functional.layer_norm(x, (x.shape[-1],), w, b, eps)


def reference_rows(x, p, heads, rotary, interleaved, qk_norm, eps=1e-5):
    """A pre-LN decoder block over one sequence's rows in float64."""
    p = {k: v.double() for k, v in p.items()}
    n, hid = x.shape
    D = hid // heads
    h = _layer_norm(x, p["norm1.weight"], p["norm1.bias"], eps)
    kvq = (h @ p["attn.query_key_value.weight"].t() + p["attn.query_key_value.bias"]).view(n, 3 * heads, D)
    k, v, q = kvq[:, :heads], kvq[:, heads:2 * heads], kvq[:, 2 * heads:]
    at = torch.arange(n)
    q = ref.norm_rotary(q, at, rotary, p["attn.query_norm"] if qk_norm else None, 1e-6, interleaved)[0]
    k = ref.norm_rotary(k, at, rotary, p["attn.key_norm"] if qk_norm else None, 1e-6, interleaved)[0]
    s = torch.einsum("qhd,khd->hqk", q, k) * D ** -0.5
    s = s.masked_fill(torch.ones(n, n).triu(1).bool(), float("-inf"))
    ctx = torch.einsum("hqk,khd->qhd", torch.softmax(s, -1), v).reshape(n, hid)
    x = x + ctx @ p["attn.dense.weight"].t() + p["attn.dense.bias"]
    h = _layer_norm(x, p["norm2.weight"], p["norm2.bias"], eps)
    h = torch.nn.functional.gelu(h @ p["mlp.dense_1.weight"].t() + p["mlp.dense_1.bias"])
    return x + h @ p["mlp.dense_2.weight"].t() + p["mlp.dense_2.bias"]


@pytest.mark.parametrize("kw", [dict(rotary_dim=64), dict(rotary_dim=32, rotary_interleaved=True, qk_norm=True), dict(qk_norm=True)])
@pytest.mark.parametrize("fused", [True, False])
def test_block_against_the_whole_sequence(kw, fused):
    """fp32 blocks (5e-4 as for the blocks without: a rotation adds a few half steps of fp32): prefill of left-padded prompts and eight steps
    across page boundaries, contiguous and paged caches bit for bit the same, against float64 recomputing every sequence."""
    _, M = _mods()
    announce("rotary block", kw, fused)
    B, S, hid, heads = 3, 37, 128, 2
    lens = [37, 9, 15]
    flat = M.Block1D(hid, heads, 4.0, dtype=F32, max_seq_len=64, fused_qkv=True, **kw).cuda()
    g = torch.Generator().manual_seed(3)
    _seed(flat, g)
    p = {k: v.detach().cpu() for k, v in flat.state_dict().items()}
    if not fused:
        split = M.Block1D(hid, heads, 4.0, dtype=F32, max_seq_len=64, fused_qkv=False, **kw).cuda()
        state = dict(p)
        for n in ("weight", "bias"):
            for name, part in zip(("key_", "value_", "query_"), state.pop(f"attn.query_key_value.{n}").chunk(3)):
                state[f"attn.{name}.{n}"] = part
        split.load_state_dict(state)
        flat = split
    paged = M.Block1D(hid, heads, 4.0, dtype=F32, max_seq_len=64, fused_qkv=fused, kv_page_size=16, **kw).cuda()
    paged.load_state_dict(flat.state_dict())
    rotary = ref.table(64, kw["rotary_dim"]) if "rotary_dim" in kw else None
    rows = [torch.randn(n, hid, generator=g) for n in lens]
    x = torch.zeros(B, S, hid)
    for b, n in enumerate(lens):
        x[b, S - n:] = rows[b]
    at = torch.tensor(lens, dtype=torch.int32).cuda()
    with torch.no_grad():
        a, b_ = flat(x.cuda(), first_cache=True, seq_lens=at), paged(x.cuda(), first_cache=True, seq_lens=at)
        assert torch.equal(a, b_)
        for step in range(9):
            for b in range(B):
                want = reference_rows(rows[b].double(), p, heads, rotary, kw.get("rotary_interleaved", False), kw.get("qk_norm", False))
                assert max_abs(a[b, -1].double().cpu(), want[-1]) <= 5e-4, (step, b)
                if step == 0:
                    assert max_abs(a[b, S - lens[b]:].double().cpu(), want) <= 5e-4, b
            new = torch.randn(B, 1, hid, generator=g)
            rows = [torch.cat((r, new[b])) for b, r in enumerate(rows)]
            x = torch.cat((x, new), 1)
            a, b_ = flat(x.cuda(), first_cache=False), paged(x.cuda(), first_cache=False)
            assert torch.equal(a, b_), step
    assert paged.attn.kv_cache.pages_in_use() == 3 + 2 + 2


@pytest.mark.parametrize("dtype,code", [(F16, torch.int8), (BF16, torch.float8_e4m3fn)])
@pytest.mark.parametrize("kw", [dict(), dict(rotary_dim=64, qk_norm=True)])
def test_attention_module_with_an_8_bit_cache(dtype, code, kw):
    """The module's steps are the operators in turn, bit for bit; native prefill of a block starts the same cache."""
    K, M = _mods()
    from energonai_amd.seqinfo import build_seq_info
    announce("8-bit module", dtype, code, kw)
    B, S, hid, heads = 3, 70, 256, 4
    lens, D = [70, 16, 31], 64
    g = torch.Generator().manual_seed(5)
    m = M.MultiHeadAttention1D(hid, heads, dtype=dtype, max_seq_len=96, kv_cache_dtype=code, kv_page_size=16, **kw).cuda()
    _seed(m, g)
    x = torch.randn(B, S, hid, generator=g).to(dtype).cuda()
    at = torch.tensor(lens, dtype=torch.int32).cuda()
    info = build_seq_info(at, B)
    with torch.no_grad():
        got = m(x, first_cache=True, seq_lens=at)
        assert type(m.kv_cache) is M.PagedKVCache8 and m.kv_cache.pages_in_use() == 5 + 1 + 2
        rows = K.depad(x, B, info, left_padded=True)
        kvq = m.query_key_value(rows).view(-1, 3 * heads, D)
        k, v, q = kvq[:, :heads], kvq[:, heads:2 * heads], kvq[:, 2 * heads:]
        how, rot = {}, None
        if kw:
            rot = K.rotary_table(96, 64, 10000.0)
            how = dict(q_weight=m.query_norm.detach(), k_weight=m.key_norm.detach())
            q, k = K.qk_norm_rotary(q, k, B, info, rot, **how)
        ctx = K.attn_fused_varlen(q, k, v, B, S, info)
        want = K.repad(m.dense(ctx.view(1, -1, hid)), B, S, info, left_padded=True)
        assert torch.equal(got, want)
        mine = list(K.kv8_pages(24, B, heads, 16, D, 6, dtype, "cuda", code))
        mine[6] = torch.arange(18, dtype=torch.int32, device="cuda").view(B, 6)
        K.kv8_pages_fill(k, v, mine, B, S, info)
        now = at.clone()
        for step in range(17):
            new = torch.randn(B, 1, hid, generator=g).to(dtype).cuda()
            x = torch.cat((x, new), 1)
            got = m(x, first_cache=False)[:, -1:]
            kvq = m.query_key_value(x[:, -1:, :]).view(B, 3 * heads, D)      # as the module has it: another stride is another library product
            q = K.kv8_pages_append(kvq[:, 2 * heads:], kvq[:, :heads], kvq[:, heads:2 * heads], mine, now.clone(), rot, **how) if kw else kvq[:, 2 * heads:]
            if not kw:
                K.kv8_pages_append(None, kvq[:, :heads], kvq[:, heads:2 * heads], mine, now.clone())
            now += 1
            want = m.dense(K.decode_attn_kv8(q, mine, now.clone()).view(B, 1, hid))
            assert torch.equal(got, want), step
        m.kv_cache.release(1)
        assert m.kv_cache.pages_in_use() == 6 + 0 + 3
        block = M.Block1D(hid, heads, 2.0, dtype=dtype, max_seq_len=96, kv_cache_dtype=code, **kw).cuda()
        plain = M.Block1D(hid, heads, 2.0, dtype=dtype, max_seq_len=96, **kw).cuda()
        _seed(block, g)
        plain.load_state_dict(block.state_dict())
        x = torch.randn(B, S, hid, generator=g).to(dtype).cuda()
        assert torch.equal(block(x, first_cache=True, seq_lens=at), plain(x, first_cache=True, seq_lens=at))
        for step in range(3):
            x = torch.cat((x, torch.randn(B, 1, hid, generator=g).to(dtype).cuda()), 1)
            a, b = block(x, first_cache=False)[:, -1].float(), plain(x, first_cache=False)[:, -1].float()
            # int8: values and keys off by 1/254 of a block's largest (e4m3: 1/16 of themselves), far under the outputs of size 1 to 3
            assert float((a - b).norm() / b.norm()) < (0.02 if code == torch.int8 else 0.1), step


def test_operators_together():
    """A server's run with grouped heads: prompts turned, attended and filled, then steps appended and attended across block and page ends, each
    context against float64 over what the cache holds."""
    K, _ = _mods()
    from energonai_amd.seqinfo import SeqInfo, build_seq_info
    from test_gpu_kv8 import check_attention
    announce("operators together")
    B, Hq, H, D, P = 4, 8, 2, 128, 32
    lens = [100, 1, 31, 64]
    for dtype, code in ((BF16, torch.int8), (F16, torch.float8_e4m3fn)):
        g = torch.Generator(device="cuda").manual_seed(2)
        T = sum(lens)
        qkv = torch.randn(T, Hq + 2 * H, D, generator=g, device="cuda", dtype=dtype)
        gains = [(1 + 0.1 * torch.randn(D, generator=g, device="cuda")).to(dtype) for _ in range(2)]
        rot = K.rotary_table(256, 64)
        how = dict(q_weight=gains[0], k_weight=gains[1])
        at = torch.tensor(lens, dtype=torch.int32, device="cuda")
        info = build_seq_info(at, B)
        q, k = K.qk_norm_rotary(qkv[:, :Hq], qkv[:, Hq:Hq + H], B, info, rot, **how)
        v = qkv[:, Hq + H:]
        spread = lambda t: t.repeat_interleave(Hq // H, 1)  # noqa: E731
        K.attn_fused_varlen(q, spread(k), spread(v), B, max(lens), info)
        cache = list(K.kv8_pages(5 * B + 1, B, H, P, D, 5, dtype, "cuda", code))
        cache[6] = torch.randperm(5 * B, generator=torch.Generator().manual_seed(1)).view(B, 5).to(torch.int32).cuda()
        K.kv8_pages_fill(k, v, cache, B, max(lens), info)
        cu = [sum(lens[:b]) for b in range(B + 1)]
        ks = [k[cu[b]:cu[b + 1]].transpose(0, 1).cpu() for b in range(B)]
        vs = [v[cu[b]:cu[b + 1]].transpose(0, 1).cpu() for b in range(B)]
        now = at.clone()
        step_info = SeqInfo(now, None, B, None, now)
        for step in range(35):
            new = torch.randn(B, Hq + 2 * H, D, generator=g, device="cuda", dtype=dtype)
            q = K.kv8_pages_append(new[:, :Hq], new[:, Hq:Hq + H], new[:, Hq + H:], cache, step_info, rot, **how)
            slot = (now % 16).tolist()
            ks = [torch.cat((ks[b], cache[4][b, :, slot[b]][:, None].cpu()), 1) for b in range(B)]
            vs = [torch.cat((vs[b], new[b, Hq + H:][:, None].cpu()), 1) for b in range(B)]
            now.add_(1)
            ctx = K.decode_attn_kv8(q, cache, step_info)
            if step % 8 == 0 or step == 34:
                check_attention(ctx, q.cpu()[:, :, None], [t.cpu() for t in cache], now.tolist(), ks, vs, code, D ** -0.5, step)


def test_native_and_general_calls_agree():
    """The same calls with lengths as a SeqInfo (one native call) and as a tensor (checked in Python) give the same bits, and refuse the same."""
    K, _ = _mods()
    from energonai_amd.seqinfo import SeqInfo, build_seq_info
    announce("native and general calls")
    B, Hq, H, D, P = 5, 6, 3, 64, 16
    lens = [0, 20, 15, 47, 3]
    g = torch.Generator(device="cuda").manual_seed(1)
    at = torch.tensor(lens, dtype=torch.int32, device="cuda")
    info, here = build_seq_info(at, B), SeqInfo(at, None, B, None, at)
    x = torch.randn(sum(lens), Hq + 2 * H, D, generator=g, device="cuda", dtype=F16)
    rot = K.rotary_table(64, 64)
    for a, b in zip(K.qk_norm_rotary(x[:, :Hq], x[:, Hq:Hq + H], B, info, rot), K.qk_norm_rotary(x[:, :Hq], x[:, Hq:Hq + H], B, at, rot)):
        assert torch.equal(a, b)
    new = x[:B]
    made = []
    for lens_ in (here, at):
        pool = torch.zeros(2, 20, H, P, D, device="cuda", dtype=F16)
        table = torch.arange(20, dtype=torch.int32, device="cuda").view(B, 4)
        q = K.kv_pages_append_rotary(new[:, :Hq], new[:, Hq:Hq + H], new[:, Hq + H:], pool[0], pool[1], lens_, table, rot)
        cache = list(K.kv8_pages(20, B, H, P, D, 4, F16, "cuda"))
        cache[6] = table
        K.kv8_pages_fill(x[:, Hq:Hq + H], x[:, Hq + H:], cache, B, 47, info if lens_ is here else at)
        q8 = K.kv8_pages_append(new[:, :Hq], new[:, Hq:Hq + H], new[:, Hq + H:], cache, lens_, rot)
        made.append([q, pool, q8, K.decode_attn_kv8(q8, cache, lens_), *K.kv8_pages_read(cache, lens_, 50)] + cache)
    assert all(torch.equal(a, b) for a, b in zip(*made))
    bad = x.float()
    for call in (lambda: K.qk_norm_rotary(bad[:, :Hq], x[:, Hq:Hq + H], B, info, rot), lambda: K.decode_attn_kv8(bad[:B, :Hq], cache, here),
                 lambda: K.kv8_pages_fill(bad[:, :H], bad[:, :H], cache, B, 47, info), lambda: K.kv8_pages_append(q8, bad[:B, :H], bad[:B, :H], cache, here, rot),
                 lambda: K.kv8_pages_read(cache[:6], here, 4), lambda: K.qk_norm_rotary(x[:, :Hq], x[:, Hq:Hq + H], B, here, rot),
                 lambda: K.qk_norm_rotary(x[:, :Hq], x[:, Hq:Hq + H], B + 1, info, rot),
                 lambda: K.kv_pages_append_rotary(new[:, :Hq], bad[:B, :H], bad[:B, :H], pool[0], pool[1], here, table, rot)):
        with pytest.raises(RuntimeError):
            call()


def test_model_refusals():
    _, M = _mods()
    for kw in (dict(rotary_dim=63), dict(rotary_dim=66), dict(rotary_dim=-2), dict(kv_cache_dtype=torch.uint8), dict(kv_cache_dtype=torch.int8, dtype=F32)):
        with pytest.raises(ValueError):
            M.MultiHeadAttention1D(128, 2, **{**dict(dtype=F16), **kw})
    with pytest.raises(ValueError):
        M.MultiHeadAttention1D(80, 2, dtype=F16, kv_cache_dtype=torch.int8)
    m = M.MultiHeadAttention1D(128, 2, dtype=F16, max_seq_len=16, rotary_dim=64, disable_past_cache=True).cuda()
    with torch.no_grad(), pytest.raises(RuntimeError, match="max_seq_len"):
        m(torch.zeros(1, 17, 128, dtype=F16, device="cuda"))
