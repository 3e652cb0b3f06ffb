"""Serving a rotary model from a cache in 8 bits, operator by operator, as a set of timed cases.

``rotary``   queries and keys of packed tokens: an RMS norm of each head, where there are gains, and the rotation by position
             in one pass (``kernel.qk_norm_rotary``);
``append``   a decode step's new rows: the same for q and k, the rotated key and the value written into a cache kept in
             16-bit (or fp32) pages (``kernel.kv_pages_append_rotary``);
``fill8``    the prompts' keys and values into a cache in 8 bits (``kernel.kv8_pages_fill``), and read back from it
             (``kernel.kv8_pages_read``);
``append8``  a decode step's new rows into that cache (``kernel.kv8_pages_append``), and the 16 positions around them read back;
``attend8``  a decode step's attention over it (``kernel.decode_attn_kv8``).

The cache in 8 bits.  A sequence's positions are taken in blocks of 16.  A block that is full lies in a page: its keys as codes
``k_pages[page, head, position, channel]``, its values as codes ``v_pages[page, head, block, channel, position in the block]``, with
one float32 scale for the block and head of each (``k_scales``, ``v_scales`` ``[page, head, block]``).  The positions behind the last
full block stay as they are in ``k_tail [sequence, head, 16, channel]`` and ``v_tail [sequence, head, channel, 16]``.  With a the largest
magnitude of a block and M the largest code (127 in int8, 448 in e4m3), ``scale = a / M`` and ``code = round(x * (M / a))``,
both in float32, to nearest even; a block whose a is under 2^-100 has scale 0 and codes 0.

Head counts, head sizes and page sizes are those of this repository's workloads and tests or generic ones beside them (grouped heads).
Activations are N(0,1), gains 1 + N(0,0.05).  The lengths of a batch follow from the case alone, their order in the batch and the pages
they lie in from the seed, so that the work of a case does not depend on the seed.
"""
from __future__ import annotations

import math
import random

import torch

own = False
BLOCK = 16
_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_LARGEST = {"int8": 127.0, "e4m3": 448.0}
_BASE = 10000.0
_EPS = 1e-6


def listed():
    return [
        # two prompts of a few tokens, 12 heads x 64: the smallest call, bound by its launch
        dict(name="rotary_few_rows_f16", op="rotary", dtype="f16", batch=2, len_lo=3, len_hi=9, len_seed=1, q_heads=12, kv_heads=12,
             head_dim=64, rotary_dim=64, interleaved=False, norm=False),
        # a ragged batch of prompts, 32 query and 8 key heads x 128 with gains
        dict(name="rotary_ragged_bf16", op="rotary", dtype="bf16", batch=7, len_lo=3, len_hi=1531, len_seed=5, q_heads=32, kv_heads=8,
             head_dim=128, rotary_dim=128, interleaved=False, norm=True),
        # four long prompts of 40 heads x 128, a quarter of each head rotated in neighbouring pairs
        dict(name="rotary_long_f16", op="rotary", dtype="f16", batch=4, len_lo=8000, len_hi=8192, len_seed=2, q_heads=40, kv_heads=40,
             head_dim=128, rotary_dim=32, interleaved=True, norm=False),
        # a small batch's decode step, 12 heads x 64
        dict(name="append_four_f16", op="append", dtype="f16", batch=4, len_lo=16, len_hi=500, len_seed=3, q_heads=12, kv_heads=12,
             head_dim=64, rotary_dim=64, interleaved=False, norm=False, page=16),
        # a large server's decode step, grouped heads with gains
        dict(name="append_256_bf16", op="append", dtype="bf16", batch=256, len_lo=1, len_hi=1000, len_seed=4, q_heads=64, kv_heads=8,
             head_dim=128, rotary_dim=128, interleaved=False, norm=True, page=64),
        # a few ragged prompts of 12 heads x 64 into the cache in int8
        dict(name="fill8_ragged_f16", op="fill8", dtype="f16", code="int8", batch=5, len_lo=9, len_hi=700, len_seed=6, kv_heads=12,
             head_dim=64, page=64),
        # eight documents of up to 16000 tokens into the cache in e4m3
        dict(name="fill8_long_bf16", op="fill8", dtype="bf16", code="e4m3", batch=8, len_lo=12000, len_hi=16000, len_seed=7, kv_heads=8,
             head_dim=128, page=128),
        # a server's decode step into the cache in int8: one sequence in 16 completes a block
        dict(name="append8_64_bf16", op="append8", dtype="bf16", code="int8", batch=64, len_lo=1, len_hi=2000, len_seed=8, q_heads=32,
             kv_heads=8, head_dim=128, rotary_dim=128, interleaved=False, norm=True, page=64),
        # interactive decoding with a short context, 12 heads x 64: launches and latency
        dict(name="attend8_one_short_f16", op="attend8", dtype="f16", code="int8", batch=1, len_lo=100, len_hi=100, len_seed=9, q_heads=12,
             kv_heads=12, head_dim=64, page=16),
        # one long document, 32 query and 8 key heads x 128
        dict(name="attend8_one_long_bf16", op="attend8", dtype="bf16", code="e4m3", batch=1, len_lo=130001, len_hi=130001, len_seed=10,
             q_heads=32, kv_heads=8, head_dim=128, page=64),
        # a server's ragged batch with a head of keys for each head of queries, 40 x 128 in int8
        dict(name="attend8_mha_f16", op="attend8", dtype="f16", code="int8", batch=16, len_lo=1, len_hi=4000, len_seed=11, q_heads=40,
             kv_heads=40, head_dim=128, page=64),
        # a large server's ragged batch, grouped heads, e4m3
        dict(name="attend8_gqa_bf16", op="attend8", dtype="bf16", code="e4m3", batch=128, len_lo=1, len_hi=8000, len_seed=12, q_heads=64,
             kv_heads=8, head_dim=128, page=64),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    kv = rng.choice([1, 2, 4, 8, 8, 12, 20, 32, 40])
    group = rng.choice([1, 1, 2, 4, 5, 7, 8, 16]) if kv <= 8 else 1
    return kv * group, kv


def _one_draw(rng):
    op = rng.choice(["rotary", "rotary", "append", "fill8", "append8", "attend8", "attend8", "attend8"])
    q_heads, kv_heads = _heads(rng)
    c = dict(op=op, kv_heads=kv_heads, head_dim=rng.choice([64, 64, 80, 96, 112, 128, 128]), len_seed=rng.randrange(1 << 20))
    if op != "fill8":
        c["q_heads"] = q_heads
    c["dtype"] = rng.choice(["f16", "bf16", "f32"] if op in ("rotary", "append") else ["f16", "bf16"])
    if op in ("rotary", "append", "append8"):
        half = c["head_dim"] // 2
        c.update(rotary_dim=2 * rng.choice([half, half, half // 2, half // 4 or 1]), interleaved=rng.random() < 0.4, norm=rng.random() < 0.5)
    if op != "rotary":
        c["page"] = rng.choice([16, 32, 64, 64, 128])
    if op in ("fill8", "append8", "attend8"):
        c["code"] = rng.choice(["int8", "e4m3"])
    c["batch"] = _log_int(rng, 1, {"rotary": 64, "append": 256, "fill8": 32, "append8": 256, "attend8": 128}[op])
    c["len_hi"] = _log_int(rng, 1, {"rotary": 8192, "append": 4000, "fill8": 16000, "append8": 4000, "attend8": 130000}[op])
    c["len_lo"] = max(1, int(c["len_hi"] * rng.choice([0.0, 0.0, 0.3, 0.75, 1.0])))
    return c


def draw(rng: random.Random):
    most = {}
    for c in listed():
        most[c["op"]] = max(most.get(c["op"], 0.0), _cost(c))
    most["append8"] = most["append"] = 4 * max(most["append"], most["append8"])
    while True:
        c = _one_draw(rng)
        if _cost(c) <= most[c["op"]]:
            return c


# ---- lengths, and what a pass cannot do without --------------------------------------------------------------------------------


def _lens(case):
    r = random.Random(case["len_seed"])
    return [r.randint(case["len_lo"], case["len_hi"]) for _ in range(case["batch"])]


def _cost(case):
    """What the plain form moves, roughly: it works on the padded batch."""
    heads = case["kv_heads"] + (case.get("q_heads", 0) if case["op"] in ("rotary", "append", "append8") else 0)
    tokens = case["batch"] * (case["len_hi"] if case["op"] in ("fill8", "attend8") else 1)
    if case["op"] == "rotary":
        tokens = sum(_lens(case))
    return float(tokens * heads * case["head_dim"])


def work(case):
    lens, D, hk, hq = _lens(case), case["head_dim"], case["kv_heads"], case.get("q_heads", 0)
    B, T, es, R = case["batch"], sum(lens), _SIZE[case["dtype"]], case.get("rotary_dim", 0)
    full = sum(n // BLOCK for n in lens)                # blocks that lie in pages
    left = T - BLOCK * full                             # positions that stay in the tails
    if case["op"] == "rotary":
        return dict(bytes=2 * T * (hq + hk) * D * es + 4 * max(lens) * R, flops=T * (hq + hk) * (3 * R + (4 * D if case["norm"] else 0)))
    if case["op"] in ("append", "append8"):
        moved = 2 * B * (hq + 2 * hk) * D * es + 4 * B * R
        flops = B * (hq + hk) * (3 * R + (4 * D if case["norm"] else 0))
        if case["op"] == "append8":
            done = sum(n % BLOCK == BLOCK - 1 for n in lens)
            moved += done * 2 * hk * (15 * D * es + BLOCK * D + 4)                       # blocks completed
            window = sum(n % BLOCK + 1 for n in lens)
            moved += 2 * hk * (window * D * es + B * BLOCK * D * es)                     # read back, padded to 16 positions
        return dict(bytes=moved, flops=flops)
    held = 2 * hk * (full * (BLOCK * D + 4) + left * D * es)                             # K and V of the cache, scales included
    if case["op"] == "fill8":
        return dict(bytes=2 * T * hk * D * es + 2 * held + 2 * B * hk * max(lens) * D * es, flops=8 * T * hk * D)
    return dict(bytes=held + 2 * B * hq * D * es, flops=4 * T * hq * D)


# ---- what a program has in hand --------------------------------------------------------------------------------------------------


def _table(rotary_dim, positions, device):
    """cos and sin of every position's angles, computed in 64 bits."""
    inv = _BASE ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * inv
    return angle.cos().float(), angle.sin().float()


def _codes(shape, code, g, dev):
    """Codes of values that are N(0,1), the block's largest near four of them."""
    x = torch.randn(shape, generator=g, device=dev, dtype=torch.float16)
    if code == "int8":
        return x.mul_(32.0).round_().clamp_(-127, 127).to(torch.int8)
    return x.mul_(112.0).clamp_(-448, 448).to(torch.float8_e4m3fn)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    lens = _lens(case)
    random.Random(seed).shuffle(lens)
    op, dtype, B = case["op"], _TYPES[case["dtype"]], case["batch"]
    D, hk, hq, T, S = case["head_dim"], case["kv_heads"], case.get("q_heads", 0), sum(lens), max(lens)
    s = dict(case=case, total=T, longest=S, full=sum(n // BLOCK for n in lens))
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    s["cu"] = torch.nn.functional.pad(s["lens"].cumsum(0, dtype=torch.int32), (1, 0))
    if op in ("rotary", "append", "append8"):
        s["rotary"] = _table(case["rotary_dim"], S + 1, dev)
        gain = lambda: (1 + 0.05 * torch.randn(D, generator=g, device=dev)).to(dtype)  # noqa: E731
        s["gains"] = (gain(), gain()) if case["norm"] else (None, None)
    if op != "attend8":
        rows = T if op in ("rotary", "fill8") else B
        heads = {"rotary": hq + hk, "fill8": 2 * hk}.get(op, hq + 2 * hk)
        x = torch.randn((rows, heads, D), generator=g, device=dev, dtype=dtype)      # a fused projection's output
        if op == "fill8":
            s["k"], s["v"] = x[:, :hk], x[:, hk:]
        else:
            s["q"], s["k"], s["v"] = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
    else:
        s["q"] = 2 * torch.randn((B, hq, 1, D), generator=g, device=dev, dtype=dtype)
    if op == "rotary":
        return s
    # pages in any order, with room for one more position
    P = case["page"]
    held = [n // P + 1 for n in lens]
    N, most = sum(held) + 3, max(held)
    ids = torch.randperm(N, generator=g, device=dev, dtype=torch.int32)
    at = torch.arange(most, device=dev) + torch.tensor([sum(held[:b]) for b in range(B)], device=dev)[:, None]
    in_use = torch.arange(most, device=dev) < torch.tensor(held, device=dev)[:, None]
    s["table"] = torch.where(in_use, ids[at.clamp(max=N - 1)], -1).contiguous()
    if op == "append":
        s["k_pool"] = torch.randn((N, hk, P, D), generator=g, device=dev, dtype=dtype)
        s["v_pool"] = torch.randn((N, hk, P, D), generator=g, device=dev, dtype=dtype)
        return s
    scale = lambda: (0.8 + 0.4 * torch.rand((N, hk, P // BLOCK), generator=g, device=dev)) / (32.0 if case["code"] == "int8" else 112.0)  # noqa: E731
    s["cache"] = (_codes((N, hk, P, D), case["code"], g, dev), _codes((N, hk, P // BLOCK, D, BLOCK), case["code"], g, dev), scale(), scale(),
                  torch.randn((B, hk, BLOCK, D), generator=g, device=dev, dtype=dtype), torch.randn((B, hk, D, BLOCK), generator=g, device=dev, dtype=dtype),
                  s["table"])
    if op == "append8":
        s["after"] = s["lens"] + 1
        s["first"] = s["lens"] // BLOCK * BLOCK
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------------------


def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    from energonai_amd import kernel as K
    from energonai_amd.seqinfo import SeqInfo
    case, B = s["case"], s["case"]["batch"]
    op = case["op"]
    info = SeqInfo(s["lens"], s["cu"], B, s["total"], s["lens"])
    if op in ("rotary", "append", "append8"):
        how = dict(q_weight=s["gains"][0], k_weight=s["gains"][1], eps=_EPS, interleaved=case["interleaved"])
    if op == "rotary":
        return K.qk_norm_rotary(s["q"], s["k"], B, info, s["rotary"], **how)
    if op == "append":
        q = K.kv_pages_append_rotary(s["q"], s["k"], s["v"], s["k_pool"], s["v_pool"], info, s["table"], s["rotary"], **how)
        return q, s["k_pool"], s["v_pool"]
    if op == "fill8":
        K.kv8_pages_fill(s["k"], s["v"], s["cache"], B, s["longest"], info)
        return K.kv8_pages_read(s["cache"], info, s["longest"])
    if op == "append8":
        q = K.kv8_pages_append(s["q"], s["k"], s["v"], s["cache"], info, s["rotary"], **how)
        k, v = K.kv8_pages_read(s["cache"], SeqInfo(s["after"], None, B, None, s["after"]), BLOCK, first=s["first"])
        return q, k, v, s["cache"][4], s["cache"][5]
    return K.decode_attn_kv8(s["q"], s["cache"], info)


def _rotated(x, gain, rotary, positions, interleaved):
    """Norm and rotation of ``[rows, heads, channels]`` in float32."""
    x = x.float()
    if gain is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * gain.float()
    cos, sin = (t[positions][:, None] for t in rotary)
    R = 2 * cos.shape[-1]
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., :R // 2], x[..., R // 2:R])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((turned, x[..., R:]), -1)


def _quantized(x, code):
    """Codes and scales of ``[blocks, heads, 16, channels]``."""
    x = x.float()
    top = x.abs().amax((-2, -1))
    some = top >= 2.0 ** -100
    largest = _LARGEST[code]
    scale = torch.where(some, top / largest, 0.0)
    y = x * torch.where(some, largest / top, 0.0)[..., None, None]
    return (y.round().to(torch.int8) if code == "int8" else y.to(torch.float8_e4m3fn).view(torch.int8)), scale


def _put_blocks(cache, code, pages, blocks, k, v):
    """Full blocks ``[n, heads, 16, channels]`` into block ``blocks[i]`` of page ``pages[i]``."""
    k_pages, v_pages, k_scales, v_scales = cache[:4]
    N, H, P, D = k_pages.shape
    ck, sk = _quantized(k, code)
    cv, sv = _quantized(v, code)
    k_pages.view(torch.int8).view(N, H, P // BLOCK, BLOCK, D)[pages, :, blocks] = ck
    v_pages.view(torch.int8)[pages, :, blocks] = cv.transpose(-1, -2)
    k_scales[pages, :, blocks] = sk
    v_scales[pages, :, blocks] = sv


def _read(cache, lens, first, S, dtype):
    """The positions ``first[b] + 0 .. S - 1`` of every sequence as ``[B, H, S, D]`` float32 pairs, zeros behind its length."""
    k_pages, v_pages, k_scales, v_scales, k_tail, v_tail, table = cache
    P = k_pages.shape[2]
    at = first[:, None] + torch.arange(S, device=lens.device)
    seq = torch.arange(len(lens), device=lens.device)[:, None]
    page = table[seq, (at // P).clamp(max=table.shape[1] - 1)].clamp(min=0).long()
    row, block, slot = at % P, at % P // BLOCK, at % BLOCK
    k = k_pages.view(torch.int8)[page, :, row].view(k_pages.dtype).float() * k_scales[page, :, block][..., None]
    v = v_pages.view(torch.int8)[page, :, block, :, slot].view(v_pages.dtype).float() * v_scales[page, :, block][..., None]
    paged = (at < lens[:, None] // BLOCK * BLOCK)[..., None, None]
    there = (at < lens[:, None])[..., None, None]
    k = torch.where(there, torch.where(paged, k, k_tail[seq, :, slot].float()), 0.0)
    v = torch.where(there, torch.where(paged, v, v_tail[seq, :, :, slot].float()), 0.0)
    return k.transpose(1, 2), v.transpose(1, 2)


def _plain(s):
    case, lens = s["case"], s["lens"].long()
    op, dtype, B = case["op"], _TYPES[case["dtype"]], case["batch"]
    dev = lens.device
    if op == "rotary":
        seq = torch.repeat_interleave(torch.arange(B, device=dev), lens, output_size=s["total"])
        at = torch.arange(s["total"], device=dev) - s["cu"].long()[seq]
        return tuple(_rotated(s[n], s["gains"][i], s["rotary"], at, case["interleaved"]).to(dtype) for i, n in enumerate("qk"))
    if op in ("append", "append8"):
        q, k = (_rotated(s[n], s["gains"][i], s["rotary"], lens, case["interleaved"]).to(dtype) for i, n in enumerate("qk"))
        page = s["table"].gather(1, lens[:, None] // case["page"])[:, 0].long()
    if op == "append":
        s["k_pool"][page, :, lens % case["page"]] = k
        s["v_pool"][page, :, lens % case["page"]] = s["v"]
        return q, s["k_pool"], s["v_pool"]
    cache = s["cache"]
    seq = torch.arange(B, device=dev)
    if op == "append8":
        cache[4][seq, :, lens % BLOCK] = k
        cache[5][seq, :, :, lens % BLOCK] = s["v"]
        # the block of every sequence is quantized; it is put into its page where it is full, and back what was there where not
        block = lens % case["page"] // BLOCK
        old = [t.view(torch.int8)[page, :, block] if t.dim() == 5 else t[page, :, block] for t in
               (cache[0].view(torch.int8).unflatten(2, (-1, BLOCK)), cache[1], cache[2], cache[3])]
        _put_blocks(cache, case["code"], page, block, cache[4], cache[5].transpose(-1, -2))
        full = lens % BLOCK == BLOCK - 1
        for t, o in zip((cache[0].view(torch.int8).unflatten(2, (-1, BLOCK)), cache[1].view(torch.int8), cache[2], cache[3]), old):
            t[page, :, block] = torch.where(full.view(-1, *[1] * (o.dim() - 1)), t[page, :, block], o)
        k, v = _read(cache, lens + 1, s["first"].long(), BLOCK, dtype)
        return q, k.to(dtype), v.to(dtype), cache[4], cache[5]
    if op == "fill8":
        cu, full = s["cu"].long(), lens // BLOCK
        owner = torch.repeat_interleave(seq, full, output_size=s["full"])
        block = torch.arange(s["full"], device=dev) - (full.cumsum(0) - full)[owner]
        rows = (cu[owner] + BLOCK * block)[:, None] + torch.arange(BLOCK, device=dev)
        page, per = s["table"][owner, BLOCK * block // case["page"]].long(), case["page"] // BLOCK
        _put_blocks(cache, case["code"], page, block % per, s["k"][rows].transpose(1, 2), s["v"][rows].transpose(1, 2))
        slot = torch.arange(BLOCK, device=dev)
        rows = (cu[:-1] + BLOCK * full)[:, None] + slot
        left = (slot < (lens % BLOCK)[:, None])[:, None, :, None]
        k, v = (x[rows.clamp(max=s["total"] - 1)].transpose(1, 2) for x in (s["k"], s["v"]))
        cache[4].copy_(torch.where(left, k, cache[4]))
        cache[5].copy_(torch.where(left, v, cache[5].transpose(-1, -2)).transpose(-1, -2))
        k, v = _read(cache, lens, torch.zeros_like(lens), s["longest"], dtype)
        return k.to(dtype), v.to(dtype)
    k, v = _read(cache, lens, torch.zeros_like(lens), s["longest"], dtype)
    H, D = case["kv_heads"], case["head_dim"]
    scores = torch.matmul(s["q"].float().view(B, H, -1, D), k.transpose(-1, -2)) * D ** -0.5
    scores = scores.masked_fill(torch.arange(s["longest"], device=dev) >= lens.view(-1, 1, 1, 1), float("-inf"))
    p = (scores - scores.amax(-1, keepdim=True)).exp()
    return (torch.matmul(p, v) / p.sum(-1, keepdim=True)).view(B, -1, 1, D).to(dtype)


# ---- the definition in 64 bits, sequence by sequence -------------------------------------------------------------------------------


def _turn64(x, gain, first, interleaved, rotary_dim):
    """``[rows, heads, channels]`` whose rows are at positions ``first`` .. in complex numbers."""
    x = x.double()
    if gain is not None:
        x = x / (x.square().mean(-1, keepdim=True) + _EPS).sqrt() * gain.double()
    R = rotary_dim
    n = torch.arange(R // 2, dtype=torch.float64, device=x.device)
    at = torch.arange(len(x), dtype=torch.float64, device=x.device) + first
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), torch.outer(at, torch.exp(-2 * n / R * math.log(_BASE))))[:, None]
    head = x[..., :R]
    pairs = head.unflatten(-1, (R // 2, 2)) if interleaved else head.unflatten(-1, (2, R // 2)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    z = z.flatten(-2) if interleaved else z.transpose(-1, -2).flatten(-2)
    return torch.cat((z, x[..., R:]), -1)


def _held64(x, code):
    """What blocks ``[.., 16, channels]`` of one head are held as."""
    top = x.double().abs().flatten(-2).max(-1).values[..., None, None]
    y = torch.where(top < 2.0 ** -100, 0.0, x.double() * (_LARGEST[code] / top))
    step = torch.ones_like(y) if code == "int8" else torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.nan_to_num((y / step).round() * step * (top / _LARGEST[code]))


def _kept64(cache, b, n):
    """Keys and values of a sequence's n positions, ``[heads, n, channels]``."""
    k_pages, v_pages, k_scales, v_scales, k_tail, v_tail, table = cache
    P, D, whole = k_pages.shape[2], k_pages.shape[3], n // BLOCK * BLOCK
    mine = table[b, :(n + P - 1) // P].long()
    k = k_pages.view(torch.int8)[mine].view(k_pages.dtype).float().double().unflatten(2, (-1, BLOCK)) * k_scales[mine].double()[..., None, None]
    v = (v_pages.view(torch.int8)[mine].view(v_pages.dtype).float().double() * v_scales[mine].double()[..., None, None]).transpose(-1, -2)
    k, v = (t.transpose(0, 1).reshape(k_pages.shape[1], -1, D)[:, :whole] for t in (k, v))
    return torch.cat((k, k_tail[b, :, :n - whole].double()), 1), torch.cat((v, v_tail[b, :, :, :n - whole].transpose(-1, -2).double()), 1)


def exact(case, seed):
    s = prepare(case, seed)
    lens, dtype, op = s["lens"].tolist(), _TYPES[case["dtype"]], case["op"]
    starts = [sum(lens[:b]) for b in range(len(lens))]
    if op == "rotary":
        return tuple(torch.cat([_turn64(s[n][t:t + m], s["gains"][i], 0, case["interleaved"], case["rotary_dim"])
                                for t, m in zip(starts, lens)]) for i, n in enumerate("qk"))
    if op in ("append", "append8"):
        q, k = (torch.cat([_turn64(s[n][b:b + 1], s["gains"][i], m, case["interleaved"], case["rotary_dim"]) for b, m in enumerate(lens)])
                for i, n in enumerate("qk"))
    if op == "append":
        pools = [s["k_pool"].double(), s["v_pool"].double()]
        for b, n in enumerate(lens):
            page = int(s["table"][b, n // case["page"]])
            pools[0][page, :, n % case["page"]] = k[b]
            pools[1][page, :, n % case["page"]] = s["v"][b].double()
        return q, *pools
    if op == "append8":
        k_tail, v_tail = s["cache"][4].double(), s["cache"][5].double()
        back = [torch.zeros(case["batch"], case["kv_heads"], BLOCK, case["head_dim"], dtype=torch.float64, device=q.device) for _ in range(2)]
        for b, n in enumerate(lens):
            m = n % BLOCK + 1
            k_tail[b, :, m - 1] = k[b].to(dtype).double()
            v_tail[b, :, :, m - 1] = s["v"][b].double()
            for t, rows in zip(back, (k_tail[b], v_tail[b].transpose(-1, -2))):
                t[b, :, :m] = _held64(rows, case["code"]) if m == BLOCK else rows[:, :m]
        return q, *back, k_tail, v_tail
    if op == "fill8":
        back = []
        for x in (s["k"], s["v"]):
            t = torch.zeros(case["batch"], case["kv_heads"], s["longest"], case["head_dim"], dtype=torch.float64, device=x.device)
            for b, n in enumerate(lens):
                rows, whole = x[starts[b]:starts[b] + n].transpose(0, 1).double(), n // BLOCK * BLOCK
                t[b, :, :whole] = _held64(rows[:, :whole].unflatten(1, (-1, BLOCK)), case["code"]).flatten(1, 2)
                t[b, :, whole:n] = rows[:, whole:]
            back.append(t)
        return tuple(back)
    out = []
    for b, n in enumerate(lens):
        k, v = _kept64(s["cache"], b, n)
        scores = s["q"][b, :, 0].double().unflatten(0, (case["kv_heads"], -1)) @ k.transpose(-1, -2) / math.sqrt(case["head_dim"])
        out.append((torch.softmax(scores, -1) @ v).flatten(0, 1)[:, None])
    return torch.stack(out)
