"""The operators of a serving step in 64 bits, one request, token or row at a time (numpy)."""
from __future__ import annotations

import math
from fractions import Fraction

import numpy as np


def cache_plan(cached, added, table, stack, free, page_size, pages, rows):
    """(seq_lens, cu_seqlens, positions, slots, free_left, table) as lists; `table` is a list of lists, not changed."""
    table = [list(row) for row in table]
    free = max(0, min(free, len(stack)))
    seq_lens, cu, positions, slots, end, asked, left = [], [0], [], [], 0, 0, free
    count = lambda n: -(-n // page_size)
    for b, (c, a) in enumerate(zip(cached, added)):
        c, a = max(c, 0), max(a, 0)
        end += a
        fits = c + a <= min(len(table[b]) * page_size, 2 ** 31 - 1) and end <= rows
        need = count(c + a) - count(c) if fits else 0
        asked += need
        served = fits and (need == 0 or asked <= free)
        if served and need:
            for j in range(need):
                table[b][count(c) + j] = stack[free - 1 - (asked - need + j)]
            left = free - asked
        for j in range(a):
            if len(slots) == rows:
                break
            page = table[b][(c + j) // page_size] if served else -1
            positions.append(min(c + j, 2 ** 31 - 1))
            slots.append(page * page_size + (c + j) % page_size if 0 <= page < pages else -1)
        seq_lens.append(c + a if served else c)
        cu.append(min(end, rows))
    behind = [-1] * (rows - len(slots))
    return seq_lens, cu, positions + behind, slots + behind, left, table


def rotate(x, cos_sin, position):
    """Rotate-half RoPE of x [heads, head_dim] at a position of the table; unchanged outside of it."""
    if not 0 <= position < len(cos_sin):
        return x
    half = x.shape[1] // 2
    cos, sin = cos_sin[position, :half], cos_sin[position, half:]
    lo, hi = x[:, :half], x[:, half:]
    return np.concatenate([lo * cos - hi * sin, hi * cos + lo * sin], 1)


def attention_decode(q, k_cache, v_cache, table, seq_lens, scale=None, softcap=0.0, window=0):
    """(out, lse, spread, reach): spread = sum p |v| / sum p, which a rounding of p scales with, reach = the largest
    scale sum_d |q_d k_d| of a head's scores, which roundings of the scores scale with."""
    batch, heads, dim = q.shape
    pages, page_size, kv_heads = k_cache.shape[:3]
    scale = scale or dim ** -0.5
    out, spread = np.zeros(q.shape), np.zeros(q.shape)
    lse, reach = np.full((batch, heads), -np.inf), np.zeros((batch, heads))
    for b in range(batch):
        end = min(max(int(seq_lens[b]), 0), table.shape[1] * page_size)
        first = max(0, end - window) if window else 0
        keys = [j for j in range(first, end) if 0 <= table[b, j // page_size] < pages]
        if not keys:
            continue
        at = np.array([table[b, j // page_size] for j in keys]), np.array([j % page_size for j in keys])
        k, v = k_cache[at], v_cache[at]  # [keys, kv_heads, dim]
        for h in range(heads):
            kv = h // (heads // kv_heads)
            with np.errstate(invalid="ignore", over="ignore"):
                s = scale * (k[:, kv] @ q[b, h])
                reach[b, h] = (scale * (np.abs(k[:, kv]) @ np.abs(q[b, h]))).max()
                if softcap:
                    s = softcap * np.tanh(s / softcap)
                if np.isnan(s).any() or (s == np.inf).any():
                    out[b, h] = lse[b, h] = np.nan
                    continue
                counts = s > -np.inf
                if not counts.any():
                    continue
                m = s.max()
                p = np.exp(s - m)
                lse[b, h] = m + math.log(p.sum())
                out[b, h] = p @ v[:, kv] / p.sum()
                spread[b, h] = p @ np.abs(v[:, kv]) / p.sum()
    return out, lse, spread, reach


def sample(z, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, logprob) of one row of logits."""
    z = np.asarray(z, dtype=np.float64)
    if np.isnan(z).any() or (z == np.inf).any() or not (z > -np.inf).any():
        return -1, math.nan
    if not temperature > 0:
        return int(z.argmax()), 0.0
    order = np.argsort(-z, kind="stable")
    d = np.full(len(z), -np.inf)
    d[z > -np.inf] = (z[z > -np.inf] - z.max()) / float(np.float32(temperature))
    # Weights as whole multiples of 2^-46 (2^-44 for more than 2^18 entries), so that sums are exact: with sums that round, equal
    # weights on both sides of a border decide by the order of additions.
    exact = 46 if len(z) <= 1 << 17 else 44
    w = np.rint(np.exp(d) * 2.0 ** exact).astype(np.int64)
    n = min(len(z), top_k) if top_k > 0 else len(z)
    upto = np.cumsum(w[order])
    limit = n
    if top_p < 1:
        share = Fraction(float(np.float32(max(top_p, 0.0)))) * int(upto[n - 1])
        limit = min(limit, int(np.searchsorted(upto, math.ceil(share))) + 1)
    if min_p > 0:
        limit = min(limit, int((np.exp(d) >= min(1.0, float(np.float32(min_p)))).sum()))
    kept = np.sort(order[:max(limit, 1)])
    upto = np.cumsum(w[kept])
    u = min(max(0.0, float(np.float32(u))), 1 - 2.0 ** -53) if u == u else 0.0
    at = int(np.searchsorted(upto, math.floor(Fraction(u) * int(upto[-1])), side="right"))
    return int(kept[at]), float(d[kept[at]] - math.log(int(upto[-1]) / 2.0 ** exact))
