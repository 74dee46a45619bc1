"""Attention over a cache of bounded size, the weights that its rows gather, and eviction: the formulas in 64 bits, a sequence and a
head at a time."""

from __future__ import annotations

import math

import torch

PAGE = 64


def rows_of(pool, table_row, kv_head, n):
    """The first n rows of a sequence in one kv head, float64 [n, dim]; pages that are not held (-1) give zeros."""
    out = torch.zeros((n, pool.shape[3]), dtype=torch.float64)
    for j in range(n):
        page = int(table_row[j // PAGE])
        if page >= 0:
            out[j] = pool[page, kv_head, j % PAGE].double()
    return out


def visible(p, n, window, first):
    j = torch.arange(n)
    seen = j <= p
    if window:
        seen &= (j > p - window) | (j < first)
    return seen


def attention(q, k_pool, v_pool, seq_start, past, counts, table, heads, kv_heads, window, first, scale, weights=None):
    """All on the CPU. Returns out [T, H, dim], lse [T, H], size [T, H, dim] (sum of softmax weight times |value|, by which rounding
    errors go), and the new weights or None (float64; rows behind a sequence's last keep what they held)."""
    T, H, dim = q.shape
    G = heads // kv_heads
    out = torch.zeros((T, H, dim), dtype=torch.float64)
    size = torch.zeros_like(out)
    lse = torch.full((T, H), -math.inf, dtype=torch.float64)
    new = None if weights is None else weights.double().clone()
    for s in range(table.shape[0]):
        c, p = int(counts[s]), int(past[s])
        n = p + c
        for k in range(kv_heads):
            keys, values = rows_of(k_pool, table[s], k, n), rows_of(v_pool, table[s], k, n)
            gained = torch.zeros(n, dtype=torch.float64)
            for i in range(c):
                t = int(seq_start[s]) + i
                see = visible(p + i, n, window, first)
                for h in range(k * G, (k + 1) * G):
                    x = keys[see] @ q[t, h].double() * scale
                    top = x.max()
                    if top == -math.inf:
                        continue
                    e = torch.exp(x - top)
                    a = e / e.sum()
                    out[t, h] = a @ values[see]
                    size[t, h] = a @ values[see].abs()
                    lse[t, h] = top + torch.log(e.sum())
                    gained[see] += a
            if new is not None and c:
                before = weights[s, k, :n].double().clone()
                before[p:] = 0
                new[s, k, :n] = before + gained
    return out, lse, size, new


def evict(weights, positions, past, length, seen, budget, first, recent):
    """One sequence and kv head: lists of (row that a place takes its contents from) and positions of the rows that stay."""
    n = length
    at = [int(positions[j]) if j < past else seen - (n - j) for j in range(n)]
    if n <= budget:
        return list(range(n)), at
    def rank(j):
        w = float(weights[j])
        safe = at[j] < first or at[j] >= seen - recent
        return (0 if safe else 1, 0 if safe else (1 if math.isnan(w) else 0), 0.0 if safe or math.isnan(w) else -w, j)
    stays = set(sorted(range(n), key=rank)[:budget])
    movers = iter(sorted(j for j in stays if j >= budget))
    source = [j if j in stays else next(movers) for j in range(budget)]
    return source, [at[j] for j in source]
