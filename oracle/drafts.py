"""Steps of drafted tokens over a paged cache, and products with 4-bit weights, restated plainly in 64 bits on the CPU (test infrastructure)."""
from __future__ import annotations

import math

import torch


def masks(parents, counts):
    """(masks, depths) of trees given as one list of parents; a parent that is no earlier node of the sequence is none."""
    out, deep, first = [], [], 0
    for n in counts:
        mine, d = [], []
        for i in range(n):
            p = parents[first + i] if i < 64 else None
            if p is None:
                mine.append(0)
                d.append(0)
                continue
            p = p if 0 <= p < i else -1
            mine.append((mine[p] if p >= 0 else 0) | 1 << i)
            d.append(d[p] + 1 if p >= 0 else 0)
        out += mine
        deep += d
        first += n
    return [m - (1 << 64) if m >> 63 else m for m in out], deep


def cached(pool, table, b, n):
    """Positions 0 .. n - 1 of sequence b, ``[heads, n, channels]``; zeros where the page is none."""
    N, H, P, D = pool.shape
    out = torch.zeros(H, n, D, dtype=torch.float64)
    for j in range(n):
        page = int(table[b, j // P])
        if 0 <= page < N:
            out[:, j] = pool[page, :, j % P].double()
    return out


def attend(q, k_new, v_new, k_pool, v_pool, lens, table, node_masks, counts, scale=None):
    """``(result, magnitude, exponent)``: the attention; sum p |v| / sum p; and the largest sum of |q k| scale of a row, elementwise or by row."""
    T, Hq, D = q.shape
    H = k_pool.shape[1]
    scale = D ** -0.5 if scale is None else scale
    out, size, most, first = torch.zeros(T, Hq, D, dtype=torch.float64), torch.zeros(T, Hq, D, dtype=torch.float64), torch.zeros(T, Hq, 1, dtype=torch.float64), 0
    for b, (n, m) in enumerate(zip(lens, counts)):
        k, v = cached(k_pool, table, b, n), cached(v_pool, table, b, n)
        for i in range(min(m, 64)):
            seen = [j for j in range(min(m, 64)) if int(node_masks[first + i]) >> j & 1]
            rows = [first + j for j in seen]
            for h in range(Hq):
                kh = torch.cat((k[h * H // Hq], k_new[rows, h * H // Hq].double()))
                vh = torch.cat((v[h * H // Hq], v_new[rows, h * H // Hq].double()))
                if not len(kh):
                    continue
                x = q[first + i, h].double()
                p = torch.softmax(kh @ x * scale, 0)
                out[first + i, h], size[first + i, h] = p @ vh, p @ vh.abs()
                most[first + i, h] = (kh.abs() @ x.abs() * scale).max()
        first += m
    return out, size, most


def accept(logits, tokens, parents, counts, max_nodes):
    path, accepted, following, first = torch.full((len(counts), max_nodes), -1, dtype=torch.int32), [], [], 0
    for b, n in enumerate(counts):
        cur, way, t = 0, [], -1
        while cur < min(n, max_nodes):
            way.append(cur)
            row = logits[first + cur].double()
            odd = row.isnan().nonzero()
            t = int(odd[0]) if len(odd) else int((row == row.max()).nonzero()[0])
            fits = [i for i in range(cur + 1, min(n, max_nodes)) if parents[first + i] == cur and tokens[first + i] == t]
            cur = fits[0] if fits else max_nodes
        path[b, :len(way)] = torch.tensor(way, dtype=torch.int32)
        accepted.append(len(way))
        following.append(t)
        first += n
    return path, torch.tensor(accepted, dtype=torch.int32), torch.tensor(following)


def extend(pool, new, lens, table, counts, path, accepted):
    """``(pool, lost)`` with the accepted rows in it."""
    pool, P, lost, first = pool.clone(), pool.shape[2], 0, 0
    for b, m in enumerate(counts):
        for i in range(min(int(accepted[b]), path.shape[1])):
            node, at = int(path[b, i]), int(lens[b]) + i
            if not 0 <= node < min(m, 64):
                continue
            page = int(table[b, at // P]) if 0 <= at < P * table.shape[1] else -1
            if 0 <= page < pool.shape[0]:
                pool[page, :, at % P] = new[first + node]
            else:
                lost += 1
        first += m
    return pool, lost


# ---- weights in 4 bits -------------------------------------------------------------------------------------------------------------


def w4_values(codes, scales, zeros, group):
    """The weight in 64 bits, and |scale| (code + zero)."""
    N, K = codes.shape[0], 2 * codes.shape[1]
    c = torch.stack((codes & 15, codes >> 4), -1).view(N, K).double()
    s = scales.double().repeat_interleave(group, 1)[:, :K]
    z = torch.full_like(c, 8.0) if zeros is None else zeros.double().repeat_interleave(group, 1)[:, :K]
    return (c - z) * s, s.abs() * (c + z)


def w4_linear(x, codes, scales, zeros, group, bias=None, act=None):
    """``(y, magnitude)``: the product; and sum |scale| (code + zero) |x| (+ |bias|), what fp32 sums of codes are accurate to."""
    w, size = w4_values(codes, scales, zeros, group)
    y, m = x.double() @ w.t(), x.double().abs() @ size.t()
    if bias is not None:
        y, m = y + bias.double(), m + bias.double().abs()
    if act == "relu":
        y = torch.where(y > 0, y, torch.zeros_like(y))
    elif act == "gelu_tanh":
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    elif act == "gelu":
        y = 0.5 * y * (1 + torch.erf(y / math.sqrt(2)))
    return y, m
