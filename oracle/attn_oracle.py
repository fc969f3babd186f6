"""CPU oracle in 64 bits for the softmax-attention operators (test infrastructure only).

    norm, rotation:  y = x / sqrt(mean(x^2) + eps) * w;  (y_a, y_b) -> (y_a c - y_b s, y_b c + y_a s)
    attention:       o_i = sum_j p_ij v_j,  p_i = softmax over j <= kv_len - q_len + i of
                     scale q_i . k_j;  a row that sees nothing is zero

``attention`` also returns sum_j p_ij |v_j|, the size that the rounding of p to bf16 is
relative to.
"""
from __future__ import annotations

import math

import torch


def norm_rope(x, weight, positions, table, *, eps=1e-6, interleaved=False):
    """x [T, H, 128] -> float64; zeros where a position lies outside the table."""
    y = x.double().clone()
    if weight is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * weight.double()
    rd = table.shape[1]
    half = rd // 2
    out = y.clone()
    for t, pos in enumerate(positions.tolist()):
        if not 0 <= pos < table.shape[0]:
            out[t] = 0
            continue
        c, s = table[pos, :half].double(), table[pos, half:].double()
        if interleaved:
            a, b = y[t, :, 0:rd:2], y[t, :, 1:rd:2]
            out[t, :, 0:rd:2], out[t, :, 1:rd:2] = a * c - b * s, b * c + a * s
        else:
            a, b = y[t, :, :half], y[t, :, half:rd]
            out[t, :, :half], out[t, :, half:rd] = a * c - b * s, b * c + a * s
    return out


def attention_one(q, k, v, scale):
    """q [R, HQ, 128], k, v [L, HK, 128]: the last R of L tokens."""
    rows, hq, d = q.shape
    length, hk = k.shape[:2]
    out = torch.zeros(rows, hq, d, dtype=torch.float64)
    size = torch.zeros(rows, hq, d, dtype=torch.float64)
    if rows == 0 or length == 0:
        return out, size
    scale = scale or 1 / math.sqrt(d)
    i = torch.arange(rows)[:, None] + (length - rows)
    seen = torch.arange(length)[None, :] <= i
    for h in range(hq):
        kh, vh = k[:, h // (hq // hk)].double(), v[:, h // (hq // hk)].double()
        z = (q[:, h].double() @ kh.T * scale).masked_fill(~seen, -math.inf)
        p = torch.nan_to_num(torch.softmax(z, dim=-1), nan=0.0)
        out[:, h], size[:, h] = p @ vh, p @ vh.abs()
    return out, size


def prefill(q, k, v, cu, scale=None):
    out = torch.zeros(q.shape, dtype=torch.float64)
    size = torch.zeros(q.shape, dtype=torch.float64)
    for a, b in zip(cu[:-1].tolist(), cu[1:].tolist()):
        out[a:b], size[a:b] = attention_one(q[a:b], k[a:b], v[a:b], scale)
    return out, size


def gather(cache, pages, length):
    """The first `length` rows of a sequence; a page outside the cache reads as zeros."""
    ps = cache.shape[1]
    rows = []
    for j in range(-(-length // ps)):
        pg = int(pages[j])
        rows.append(cache[pg] if 0 <= pg < cache.shape[0] else torch.zeros_like(cache[0]))
    return (torch.cat(rows) if rows else cache[0][:0])[:length]


def paged(q, k_cache, v_cache, block_table, kv_lens, cu, scale=None):
    """q [T, HQ, 128] packed by cu."""
    out = torch.zeros(q.shape, dtype=torch.float64)
    size = torch.zeros(q.shape, dtype=torch.float64)
    most = block_table.shape[1] * k_cache.shape[1]
    for n, (a, b) in enumerate(zip(cu[:-1].tolist(), cu[1:].tolist())):
        length = min(max(int(kv_lens[n]), 0), most)
        k = gather(k_cache, block_table[n], length)
        v = gather(v_cache, block_table[n], length)
        skip = min(max(b - a - length, 0), b - a)  # rows before the first cached token
        if b > a + skip:
            out[a + skip:b], size[a + skip:b] = attention_one(q[a + skip:b], k, v, scale)
    return out, size
