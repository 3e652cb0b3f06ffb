"""Plain restatement, on the CPU and in 64 bits where numbers are computed, of norm and rotation of heads and of the K/V cache in 8 bits."""
from __future__ import annotations

import math

import torch

BLOCK = 16
LARGEST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def table(positions, rotary_dim, base=10000.0):
    """cos and sin as float32, angle by angle."""
    cos = torch.empty(positions, rotary_dim // 2)
    sin = torch.empty(positions, rotary_dim // 2)
    for i in range(rotary_dim // 2):
        inv = base ** (-2.0 * i / rotary_dim)
        for p in range(positions):
            cos[p, i], sin[p, i] = math.cos(p * inv), math.sin(p * inv)
    return cos, sin


def norm_rotary(x, positions, rotary, weight, eps, interleaved):
    """``[rows, heads, D]`` in float64: (y, the magnitude its rounding errors scale with)."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    y, size = x.clone(), x.abs()
    if rotary is not None:
        cos, sin = (t.double()[positions][:, None, :] for t in rotary)
        n = cos.shape[-1]
        ia = torch.arange(n) * 2 if interleaved else torch.arange(n)
        ib = ia + 1 if interleaved else ia + n
        a, b = x[..., ia], x[..., ib]
        y[..., ia] = a * cos - b * sin
        y[..., ib] = b * cos + a * sin
        size[..., ia] = size[..., ib] = a.abs() + b.abs()
    return y, size


def quantize(block, code_dtype):
    """One ``[16, D]`` block of one head: (codes ``[16, D]``, scale), the float32 definition."""
    x = block.float()
    top = x.abs().max()
    if not torch.isfinite(x).all():
        return torch.zeros_like(x).to(code_dtype), torch.tensor(float("nan"))
    if top < 2.0 ** -100:
        return torch.zeros_like(x).to(code_dtype), torch.tensor(0.0)
    m = torch.tensor(LARGEST[code_dtype])
    y = x * (m / top)
    return (y.round() if code_dtype == torch.int8 else y).to(code_dtype), top / m


class Cache:
    """Sequences as rows in 16 bits, [H, n, D] for keys and values, and what a cache in 8 bits holds of them."""

    def __init__(self, heads, D, code_dtype):
        self.heads, self.D, self.code = heads, D, code_dtype

    def held(self, rows):
        """Float64 values of ``[H, n, D]`` rows as the cache stands for them."""
        out = rows.double().clone()
        n = rows.shape[1]
        for h in range(rows.shape[0]):
            for j in range(n // BLOCK):
                c, s = quantize(rows[h, j * BLOCK:(j + 1) * BLOCK], self.code)
                out[h, j * BLOCK:(j + 1) * BLOCK] = c.float().double() * s.double()
        return out


def put(cache, b, k, v):
    """Writes sequence b's ``[H, n, D]`` rows into the CPU tensors of a cache, through its page table."""
    k_pages, v_pages, k_scales, v_scales, k_tail, v_tail, page_table = cache
    H, n, _ = k.shape
    P, N = k_pages.shape[2], k_pages.shape[0]
    for h in range(H):
        for j in range(n // BLOCK):
            pid = int(page_table[b, j * BLOCK // P])
            if not 0 <= pid < N:
                continue
            r = j * BLOCK % P
            rows = slice(j * BLOCK, (j + 1) * BLOCK)
            kc, ks = quantize(k[h, rows], k_pages.dtype)
            vc, vs = quantize(v[h, rows], v_pages.dtype)
            k_pages.view(torch.int8)[pid, h, r:r + BLOCK] = kc.view(torch.int8)
            v_pages.view(torch.int8)[pid, h, r // BLOCK] = vc.view(torch.int8).t()
            k_scales[pid, h, r // BLOCK] = ks
            v_scales[pid, h, r // BLOCK] = vs
    m = n % BLOCK
    k_tail[b, :, :m] = k[:, n - m:]
    v_tail[b, :, :, :m] = v[:, n - m:].transpose(1, 2)


def attention(q, k, v, scale):
    """One query ``[G, D]`` a row over float64 ``[n, D]`` keys and values of a head: (context, sum of |p v|, the errors' measure)."""
    if k.shape[0] == 0:
        return torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64)
    p = torch.softmax(q.double() @ k.t() * scale, -1)
    return p @ v, p @ v.abs()
