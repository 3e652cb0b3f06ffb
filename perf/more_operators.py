"""Decoding with drafted tokens on weights of 4 bits, operator by operator, as a set of timed cases.

A step of such a program has several tokens a sequence: the newest one, which is certain, and tokens that a cheap model drafted behind
it.  They form a tree (node 0 is its root, a node's parent comes before it), and one pass over cache and weights checks them all.

``w4``      rows times a weight of 4 bits: ``y = act(x W^T + b)``, ``W[n, k] = (code - zero[n, g]) * scale[n, g]`` with one scale (and zero
            point; without them 8) for each group g of neighbouring channels (``kernel.linear_w4``);
``tree``    attention of the nodes over a paged cache and over one another: a node sees its sequence's cached positions and the nodes of
            its mask, those on its way from the root (``kernel.decode_attn_tree``), grouped heads;
``accept``  the nodes that a greedy decoding would have chosen: from the root to the child whose token has the largest logit, as long
            as there is one, and the token behind the last (``kernel.accept_drafts``);
``extend``  the accepted nodes' keys and values into the pages (``kernel.kv_pages_extend``).

Widths, head counts, head sizes and page sizes are those of this repository's workloads and tests or generic ones beside them.  Lengths, trees
and what is accepted follow from the case alone; their order in the batch, the pages, tokens and values follow from the seed.
Activations are N(0,1); codes spread as those of normal weights.
"""
from __future__ import annotations

import math
import random

import torch

own = False
_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
MOST_NODES = 64


def listed():
    return [
        # the smallest projection, one sequence without drafts: launch and latency
        dict(name="w4_one_row_small_f16", op="w4", dtype="f16", rows=1, width=768, out=2304, group=64, zeros=False, bias=True, act="none"),
        # one sequence, the widest projection of a large model: the stream of the codes
        dict(name="w4_one_row_wide_bf16", op="w4", dtype="bf16", rows=1, width=7168, out=28672, group=128, zeros=True, bias=False, act="none"),
        # the drafted nodes of a few sequences together
        dict(name="w4_drafts_f16", op="w4", dtype="f16", rows=40, width=9216, out=9216, group=128, zeros=False, bias=True, act="none"),
        # prompts through the same weights, small groups, an output that fills no tile
        dict(name="w4_prompt_bf16", op="w4", dtype="bf16", rows=2000, width=5120, out=13841, group=32, zeros=True, bias=True, act="relu"),
        # interactive decoding with a short context: a few nodes, 12 heads x 64
        dict(name="tree_one_short_f16", op="tree", dtype="f16", batch=1, len_lo=100, len_hi=100, nodes_lo=8, nodes_hi=8, case_seed=1,
             q_heads=12, kv_heads=12, head_dim=64, page=16),
        # a server's ragged batch, grouped heads, small trees
        dict(name="tree_server_bf16", op="tree", dtype="bf16", batch=24, len_lo=1, len_hi=4000, nodes_lo=1, nodes_hi=16, case_seed=2,
             q_heads=32, kv_heads=8, head_dim=128, page=64),
        # large trees, a head of keys for each head of queries
        dict(name="tree_mha_f16", op="tree", dtype="f16", batch=16, len_lo=500, len_hi=2000, nodes_lo=24, nodes_hi=64, case_seed=3,
             q_heads=56, kv_heads=56, head_dim=128, page=64),
        # one long document, a large tree, eight heads of queries a head of keys
        dict(name="tree_long_bf16", op="tree", dtype="bf16", batch=1, len_lo=130001, len_hi=130001, nodes_lo=63, nodes_hi=63, case_seed=4,
             q_heads=64, kv_heads=8, head_dim=128, page=64),
        # one tree, a vocabulary whose rows lie at any address
        dict(name="accept_one_f16", op="accept", dtype="f16", batch=1, nodes_lo=24, nodes_hi=24, case_seed=5, vocab=50257),
        # a server's trees over a large vocabulary
        dict(name="accept_64_bf16", op="accept", dtype="bf16", batch=64, nodes_lo=1, nodes_hi=64, case_seed=6, vocab=128000),
        # a small batch's accepted rows, 12 heads x 64
        dict(name="extend_four_f16", op="extend", dtype="f16", batch=4, len_lo=16, len_hi=500, nodes_lo=4, nodes_hi=16, case_seed=7,
             kv_heads=12, head_dim=64, page=16),
        # a large server's
        dict(name="extend_256_bf16", op="extend", dtype="bf16", batch=256, len_lo=1, len_hi=1000, nodes_lo=1, nodes_hi=32, case_seed=8,
             kv_heads=8, head_dim=128, page=64),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _one_draw(rng):
    op = rng.choice(["w4", "w4", "w4", "tree", "tree", "tree", "accept", "extend"])
    c = dict(op=op, dtype=rng.choice(["f16", "bf16"]))
    if op == "w4":
        c.update(rows=_log_int(rng, 1, 2000), width=8 * _log_int(rng, 4, 2048), out=_log_int(rng, 1, 30000), group=rng.choice([32, 64, 128, 128]),
                 zeros=rng.random() < 0.5, bias=rng.random() < 0.5, act=rng.choice(["none", "none", "relu", "gelu_tanh"]))
        return c
    c["batch"] = _log_int(rng, 1, {"tree": 64, "accept": 64, "extend": 256}[op])
    c["nodes_hi"] = _log_int(rng, 1, MOST_NODES)
    c["nodes_lo"] = max(1, int(c["nodes_hi"] * rng.choice([0.0, 0.3, 1.0])))
    c["case_seed"] = rng.randrange(1 << 20)
    if op == "accept":
        c["dtype"] = rng.choice(["f16", "bf16", "f32"])
        c["vocab"] = _log_int(rng, 100, 130000)
        return c
    kv = rng.choice([1, 2, 4, 8, 8, 12, 20, 32, 40])
    c.update(kv_heads=kv, head_dim=rng.choice([64, 64, 72, 80, 96, 112, 128, 128]), page=rng.choice([16, 32, 64, 64, 128]))
    c["len_hi"] = _log_int(rng, 1, 130000 if op == "tree" else 4000)
    c["len_lo"] = int(c["len_hi"] * rng.choice([0.0, 0.0, 0.3, 0.75, 1.0]))
    if op == "tree":
        c["q_heads"] = kv * (rng.choice([1, 1, 2, 4, 5, 7, 8, 16]) if kv <= 8 else 1)
    else:
        c["dtype"] = rng.choice(["f16", "bf16", "f32"])
    return c


def draw(rng: random.Random):
    most = {}
    for c in listed():
        most[c["op"]] = tuple(max(a, b) for a, b in zip(most.get(c["op"], (0.0, 0.0)), _cost(c)))
    while True:
        c = _one_draw(rng)
        if all(a <= b for a, b in zip(_cost(c), most[c["op"]])):
            return c


# ---- lengths and trees, and what a pass cannot do without ------------------------------------------------------------------------


def _sizes(case):
    """Context length and nodes of each sequence."""
    r = random.Random(case["case_seed"])
    return [(r.randint(case.get("len_lo", 0), case.get("len_hi", 0)), r.randint(case["nodes_lo"], case["nodes_hi"])) for _ in range(case["batch"])]


def _trees(case):
    """Parents of each sequence's nodes (-1: the root), and the way that is accepted, from the root."""
    r = random.Random(case["case_seed"] + 1)
    trees = []
    for _, n in _sizes(case):
        parents = [-1] + [r.randint(max(0, i - 4), i - 1) for i in range(1, n)]
        way, goes_on = [0], True
        while goes_on:
            children = [i for i in range(n) if parents[i] == way[-1]]
            goes_on = bool(children) and r.random() < 0.75
            if goes_on:
                way.append(r.choice(children))
        trees.append((parents, way))
    return trees


def _cost(case):
    """What the plain form moves and computes, roughly."""
    if case["op"] == "w4":
        return float(case["width"] * case["out"] + 8 * case["rows"] * case["out"]), float(case["rows"] * case["width"] * case["out"])
    sizes = _sizes(case)
    if case["op"] == "tree":
        return (float(sum(n + m for n, m in sizes) * case["kv_heads"] * case["head_dim"]),
                float(sum((n + m) * m for n, m in sizes) * case["q_heads"] * case["head_dim"]))
    if case["op"] == "accept":
        return float(sum(m for _, m in sizes) * case["vocab"] * _SIZE[case["dtype"]]), 0.0
    return float(sum(n + m for n, m in sizes) * case["kv_heads"] * case["head_dim"] * _SIZE[case["dtype"]]), 0.0


def work(case):
    es = _SIZE[case["dtype"]]
    if case["op"] == "w4":
        R, K, N, groups = case["rows"], case["width"], case["out"], -(-case["width"] // case["group"])
        return dict(bytes=N * K // 2 + N * groups * (es + (1 if case["zeros"] else 0)) + R * K * es + R * N * es + (N * es if case["bias"] else 0),
                    flops=2 * R * K * N)
    sizes = _sizes(case)
    nodes = sum(m for _, m in sizes)
    if case["op"] == "accept":
        return dict(bytes=sum(len(way) for _, way in _trees(case)) * case["vocab"] * es + 12 * nodes, flops=0)
    hk, D = case["kv_heads"], case["head_dim"]
    if case["op"] == "extend":
        return dict(bytes=2 * 2 * sum(len(way) for _, way in _trees(case)) * hk * D * es, flops=0)
    hq = case["q_heads"]
    seen = 0
    for (n, m), (parents, _) in zip(sizes, _trees(case)):
        depth = []
        for p in parents:
            depth.append(1 if p < 0 else depth[p] + 1)
        seen += n * m + sum(depth)
    return dict(bytes=2 * sum(n + m for n, m in sizes) * hk * D * es + 2 * nodes * hq * D * es + 8 * nodes, flops=4 * seen * hq * D)


# ---- what a program has in hand --------------------------------------------------------------------------------------------------


def _prepare_w4(case, g, dev, s):
    R, K, N, dtype = case["rows"], case["width"], case["out"], _TYPES[case["dtype"]]
    groups = -(-K // case["group"])

    def code():      # two a byte, of weights that are N(0,1) with a step of 0.37
        return torch.randn((N, K // 2), generator=g, device=dev, dtype=torch.float16).mul_(2.7).round_().clamp_(-8, 7).to(torch.int8)

    s["codes"] = ((code() + 8) | ((code() + 8) << 4)).view(torch.uint8)
    s["scales"] = ((0.6 + 0.8 * torch.rand((N, groups), generator=g, device=dev)) * 0.37 / math.sqrt(K)).to(dtype)
    s["zeros"] = torch.randint(6, 11, (N, groups), generator=g, device=dev, dtype=torch.uint8) if case["zeros"] else None
    s["x"] = torch.randn((1, R, K), generator=g, device=dev, dtype=dtype)
    s["bias"] = torch.randn(N, generator=g, device=dev, dtype=dtype) if case["bias"] else None
    if own:
        from energonai_amd import kernel as K4
        s["weight"] = K4.w4_weight(s["codes"], s["scales"], s["zeros"], group_size=case["group"])


def _pages(lens, extra, case, g, dev, s):
    """Pools and a table, pages in any order, with room for the new positions."""
    P, hk, D, dtype = case["page"], case["kv_heads"], case["head_dim"], _TYPES[case["dtype"]]
    held = [(n + m + P - 1) // P for n, m in zip(lens, extra)]
    N, most = sum(held) + 3, max(max(held), 1)
    ids = torch.randperm(N, generator=g, device=dev, dtype=torch.int32)
    at = torch.arange(most, device=dev) + torch.tensor([sum(held[:b]) for b in range(len(held))], device=dev)[:, None]
    in_use = torch.arange(most, device=dev) < torch.tensor(held, device=dev)[:, None]
    s["table"] = torch.where(in_use, ids[at.clamp(max=N - 1)], -1).contiguous()
    s["k_pool"] = torch.randn((N, hk, P, D), generator=g, device=dev, dtype=dtype)
    s["v_pool"] = torch.randn((N, hk, P, D), generator=g, device=dev, dtype=dtype)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    s = dict(case=case)
    if case["op"] == "w4":
        _prepare_w4(case, g, dev, s)
        return s
    both = list(zip(_sizes(case), _trees(case)))
    random.Random(seed).shuffle(both)
    lens, nodes = [n for (n, _), _ in both], [m for (_, m), _ in both]
    parents, ways = [p for _, (p, _) in both], [w for _, (_, w) in both]
    B, T, dtype = case["batch"], sum(nodes), _TYPES[case["dtype"]]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    s.update(lens_host=lens, nodes_host=nodes, longest=max(nodes))
    s["lens"], s["nodes"], s["parents"] = i32(lens), i32(nodes), i32([p for one in parents for p in one])
    s["cu"] = torch.nn.functional.pad(s["nodes"].cumsum(0, dtype=torch.int32), (1, 0))
    masks, depths = [], []
    for one in parents:
        mine, deep = [], []
        for i, p in enumerate(one):
            mine.append((mine[p] if p >= 0 else 0) | 1 << i)
            deep.append(deep[p] + 1 if p >= 0 else 0)
        masks += [m - (1 << 64) if m >> 63 else m for m in mine]
        depths += deep
    s["masks"], s["depths"] = torch.tensor(masks, dtype=torch.int64, device=dev), i32(depths)
    if case["op"] == "accept":
        V = case["vocab"]
        s["tokens"] = torch.randint(0, V, (T,), generator=g, device=dev)
        logits = torch.randn((T, V), generator=g, device=dev, dtype=dtype)
        first, rows, children, stops = 0, [], [], []
        for way, m in zip(ways, nodes):
            rows += [first + i for i in way[:-1]]
            children += [first + i for i in way[1:]]
            stops.append(first + way[-1])
            first += m
        if rows:
            logits[torch.tensor(rows, device=dev), s["tokens"][torch.tensor(children, device=dev)]] = 12.0
        # the last accepted node's choice is none of its children's tokens, as far as there are others
        logits[torch.tensor(stops, device=dev), torch.randint(0, V, (B,), generator=g, device=dev)] = 11.0
        s["logits"] = logits
        return s
    _pages(lens, nodes, case, g, dev, s)
    hk, D = case["kv_heads"], case["head_dim"]
    if case["op"] == "tree":
        hq = case["q_heads"]
        x = torch.randn((T, hq + 2 * hk, D), generator=g, device=dev, dtype=dtype)      # a fused projection's output
        s["q"], s["k"], s["v"] = 1.5 * x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
        return s
    x = torch.randn((T, 2 * hk, D), generator=g, device=dev, dtype=dtype)
    s["k"], s["v"] = x[:, :hk], x[:, hk:]
    s["path"] = i32([w + [-1] * (s["longest"] - len(w)) for w in ways])
    s["counts"] = i32([len(w) for w in ways])
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------------------


def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    from energonai_amd import kernel as K
    from energonai_amd.seqinfo import SeqInfo
    case = s["case"]
    if case["op"] == "w4":
        return K.linear_w4(s["x"], s["weight"], bias=s["bias"], activation=case["act"])
    B = case["batch"]
    tree = K.DraftTree(s["parents"], s["masks"], s["depths"], SeqInfo(s["nodes"], s["cu"], B, len(s["masks"]), s["nodes"]), s["longest"])
    if case["op"] == "accept":
        return K.accept_drafts(s["logits"], s["tokens"], tree)
    cached = SeqInfo(s["lens"], None, B, None, s["lens"])
    if case["op"] == "tree":
        return K.decode_attn_tree(s["q"], s["k"], s["v"], s["k_pool"], s["v_pool"], cached, s["table"], tree)
    K.kv_pages_extend(s["k"], s["v"], s["k_pool"], s["v_pool"], cached, s["table"], tree, s["path"], s["counts"])
    return s["k_pool"], s["v_pool"]


def _activated(y, act):
    if act == "relu":
        return y.clamp(min=0)
    if act == "gelu_tanh":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    return y


def _plain(s):
    case = s["case"]
    dtype, op = _TYPES[case["dtype"]], case["op"]
    if op == "w4":
        N, K = case["out"], case["width"]
        c = torch.stack((s["codes"] & 15, s["codes"] >> 4), -1).view(N, K).float()
        by = s["scales"].float().repeat_interleave(case["group"], 1)[:, :K]
        zero = 8.0 if s["zeros"] is None else s["zeros"].float().repeat_interleave(case["group"], 1)[:, :K]
        y = torch.matmul(s["x"].float(), ((c - zero) * by).t())
        return _activated(y if s["bias"] is None else y + s["bias"].float(), case["act"]).to(dtype)
    if op == "accept":
        return _plain_accept(s)
    if op == "extend":
        B, P, longest = case["batch"], case["page"], s["longest"]
        seq = torch.arange(B, device=s["lens"].device)[:, None]
        step = torch.arange(longest, device=s["lens"].device)
        there = step < s["counts"][:, None]
        at = (s["lens"][:, None] + step).long()
        page = s["table"][seq, (at // P).clamp(max=s["table"].shape[1] - 1)].long()
        row = (s["cu"][:-1, None] + s["path"]).long()
        # steps that are none write the sequence's first new row once more
        page, slot, row = (torch.where(there, t, t[:, :1]) for t in (page, at % P, row))
        s["k_pool"][page, :, slot] = s["k"][row]
        s["v_pool"][page, :, slot] = s["v"][row]
        return s["k_pool"], s["v_pool"]
    hk, D, P, first, out = case["kv_heads"], case["head_dim"], case["page"], 0, []
    for b, (n, m) in enumerate(zip(s["lens_host"], s["nodes_host"])):
        mine = s["table"][b, :(n + P - 1) // P].long()
        rows = slice(first, first + m)
        k, v = (torch.cat((pool[mine].transpose(0, 1).reshape(hk, -1, D)[:, :n], new[rows].transpose(0, 1)), 1).float()
                for pool, new in ((s["k_pool"], s["k"]), (s["v_pool"], s["v"])))
        q = s["q"][rows].float().view(m, hk, -1, D).permute(1, 2, 0, 3).reshape(hk, -1, D)          # group by group, node by node
        scores = torch.matmul(q, k.transpose(-1, -2).contiguous()) * D ** -0.5
        seen = (s["masks"][rows, None] >> torch.arange(m, device=k.device)) & 1
        scores.view(hk, -1, m, n + m)[..., n:].masked_fill_(seen == 0, float("-inf"))
        p = (scores - scores.amax(-1, keepdim=True)).exp()
        o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
        out.append(o.view(hk, -1, m, D).permute(2, 0, 1, 3).reshape(m, -1, D).to(dtype))
        first += m
    return torch.cat(out)


def _plain_accept(s):
    B, longest, V, dev = s["case"]["batch"], s["longest"], s["case"]["vocab"], s["logits"].device
    T = len(s["parents"])
    most = s["logits"].amax(1, keepdim=True)
    choice = torch.where(s["logits"] == most, torch.arange(V, device=dev), V).amin(1)
    # nodes of every sequence, padded
    step = torch.arange(longest, device=dev)
    at = (s["cu"][:-1, None] + step).clamp(max=T - 1).long()
    there = step < s["nodes"][:, None]
    parents, tokens = torch.where(there, s["parents"][at].long(), -2), s["tokens"][at]
    choice = choice[at]
    seq = torch.arange(B, device=dev)
    cur, goes_on = torch.zeros(B, dtype=torch.long, device=dev), torch.ones(B, dtype=torch.bool, device=dev)
    path = torch.full((B, longest), -1, dtype=torch.int32, device=dev)
    path[:, 0] = 0
    count = torch.ones(B, dtype=torch.int32, device=dev)
    for i in range(1, longest):
        fits = (parents == cur[:, None]) & (tokens == choice[seq, cur][:, None])
        child = torch.where(fits, step, longest).amin(1)
        goes_on = goes_on & (child < longest)
        cur = torch.where(goes_on, child, cur)
        path[:, i] = torch.where(goes_on, child, -1)
        count += goes_on
    return path, count, choice[seq, cur]


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "w4":
        N, K, G = case["out"], case["width"], case["group"]
        y = torch.zeros((case["rows"], N), dtype=torch.float64, device=s["x"].device)
        for g in range(-(-K // G)):
            lo, hi = g * G, min(K, (g + 1) * G)
            byte = s["codes"][:, lo // 2:hi // 2].long()
            c = torch.empty((N, hi - lo), dtype=torch.float64, device=byte.device)
            c[:, 0::2] = (byte % 16).double()
            c[:, 1::2] = (byte // 16).double()
            c -= 8.0 if s["zeros"] is None else s["zeros"][:, g:g + 1].double()
            y += (s["x"][0, :, lo:hi].double() @ c.t()) * s["scales"][:, g].double()
        if s["bias"] is not None:
            y += s["bias"].double()
        if case["act"] == "relu":
            y = torch.where(y > 0, y, 0.0)
        elif case["act"] == "gelu_tanh":
            z = 2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)
            y = y * torch.sigmoid(z)
        return y[None]
    if case["op"] == "accept":
        path = torch.full((case["batch"], s["longest"]), -1, dtype=torch.int32)
        counts, last, first = [], [], 0
        parents, tokens = s["parents"].tolist(), s["tokens"].tolist()
        for b, m in enumerate(s["nodes_host"]):
            cur, way = 0, [0]
            while True:
                row = s["logits"][first + cur].double()
                t = int((row == row.max()).nonzero()[0])
                fits = [i for i in range(m) if parents[first + i] == cur and tokens[first + i] == t]
                if not fits:
                    break
                cur = fits[0]
                way.append(cur)
            path[b, :len(way)] = torch.tensor(way, dtype=torch.int32)
            counts.append(len(way))
            last.append(t)
            first += m
        dev = s["logits"].device
        return path.to(dev), torch.tensor(counts, dtype=torch.int32, device=dev), torch.tensor(last, device=dev)
    lens, nodes, P = s["lens_host"], s["nodes_host"], case["page"]
    if case["op"] == "extend":
        pools, first = [s["k_pool"].double(), s["v_pool"].double()], 0
        table, path = s["table"].tolist(), s["path"].tolist()
        for b, (n, m) in enumerate(zip(lens, nodes)):
            for i, node in enumerate(path[b][:int(s["counts"][b])]):
                for pool, new in zip(pools, (s["k"], s["v"])):
                    pool[table[b][(n + i) // P], :, (n + i) % P] = new[first + node].double()
            first += m
        return tuple(pools)
    hk, hq, D, first, out = case["kv_heads"], case["q_heads"], case["head_dim"], 0, []
    for b, (n, m) in enumerate(zip(lens, nodes)):
        ids = s["table"][b, :-(-n // P)].long()
        seen = torch.tensor([[bool(w >> i & 1) for i in range(m)] for w in s["masks"][first:first + m].tolist()], device=s["q"].device)
        o = torch.empty((m, hq, D), dtype=torch.float64, device=s["q"].device)
        for h in range(hk):
            k, v = (torch.cat((pool[ids, h].reshape(-1, D)[:n], new[first:first + m, h])).double()
                    for pool, new in ((s["k_pool"], s["k"]), (s["v_pool"], s["v"])))
            for j in range(h * hq // hk, (h + 1) * hq // hk):
                scores = s["q"][first:first + m, j].double() @ k.t() / math.sqrt(D)
                scores[:, n:][~seen] = -math.inf
                o[:, j] = torch.softmax(scores, 1) @ v
        out.append(o)
        first += m
    return torch.cat(out)
