"""Drafted tokens: what nodes see, attention over a tree, verification and compaction: the definitions in 64 bits, a sequence at a time."""

from __future__ import annotations

import math

import torch

PAGE = 64


def ways(parents, window=0):
    """Per node the list of nodes that it sees (itself first, then up), and its depth."""
    seen, depth = [], []
    for i, p in enumerate(parents):
        up = p if 0 <= p < i else -1
        depth.append(0 if up < 0 else depth[up] + 1)
        way, j = [], i
        while j >= 0:
            way.append(j)
            j = parents[j] if 0 <= parents[j] < j else -1
        seen.append(way[:window] if window else way)
    return seen, depth


def bits(seen, words):
    out = torch.zeros((len(seen), words), dtype=torch.int64)
    for i, way in enumerate(seen):
        for j in way:
            out[i, j // 32] |= 1 << (j % 32)
    return torch.where(out >= 1 << 31, out - (1 << 32), out).to(torch.int32)


def attention(q, k_pool, v_pool, seq_start, past, counts, seen_bits, positions, table, heads, kv_heads, window, scale):
    """All on the CPU. Returns out [T, H, dim], size [T, H, dim] (sum of softmax weight times |value|) and slack [T, H]: the largest
    relative error of a weight that 32-bit sums of products and of weights may leave."""
    T, H, dim = q.shape
    G = heads // kv_heads
    out = torch.zeros((T, H, dim), dtype=torch.float64)
    size, slack = torch.zeros_like(out), torch.zeros((T, H), dtype=torch.float64)
    for s in range(table.shape[0]):
        p, c = int(past[s]), int(counts[s])
        for i in range(c):
            t = int(seq_start[s]) + i
            lo = max(0, int(positions[t]) - window + 1) if window else 0
            rows = list(range(lo, p)) + [p + b for b in range(c) if int(seen_bits[t, b // 32]) >> (b % 32) & 1]
            if not rows:
                continue
            at = torch.tensor(rows)
            pages = table[s][at // PAGE].long()
            assert bool((pages >= 0).all())
            for k in range(kv_heads):
                keys, values = k_pool[pages, k, at % PAGE].double(), v_pool[pages, k, at % PAGE].double()
                for h in range(k * G, (k + 1) * G):
                    x = keys @ q[t, h].double() * scale
                    if float(x.max()) == -math.inf:
                        continue
                    a = torch.softmax(x, 0)
                    out[t, h], size[t, h] = a @ values, a @ values.abs()
                    # a score is a sum of dim products, each step off by half of 2^-23 of what it adds up; so are the exponent that becomes a
                    # power (by a part of the scores' size) and the sums over the keys
                    reach = float((keys.abs() @ q[t, h].double().abs() * scale).max())
                    slack[t, h] = 2.0 ** -24 * (2 * (dim + 8) * reach + 2 * len(rows) + 16)
    return out, size, slack


def verify(logits, tokens, parents, uniforms, temperature, limit, probs=None, floors=None):
    """One sequence: (path, chosen). Rows of this sequence alone."""
    count = logits.shape[0]
    if count == 0:
        return [], -1
    node, path = 0, [0]
    while True:
        row = logits[node, :limit].double()
        row = torch.where(torch.isnan(row), torch.full_like(row, -math.inf), row)
        children = [j for j in range(node + 1, count) if int(parents[j]) == node]
        if temperature <= 0:
            best = int((row == row.max()).nonzero()[0])
            nxt = [j for j in children if int(tokens[j]) == best]
            if not nxt:
                return path, best
            node = nxt[0]
            path.append(node)
            continue
        if floors is not None:
            row = torch.where(row >= float(floors[node]), row, torch.full_like(row, -math.inf))
        top = row.max()
        if float(top) == -math.inf:
            return path, 0
        p = torch.where(row == top, torch.ones_like(row), torch.exp((row - (top if math.isfinite(top) else 0.0)) / temperature) if math.isfinite(top) else torch.zeros_like(row))
        p = p / p.sum()
        whole, taken = p.clone(), None
        q = None if probs is None else probs[node, :limit].double()
        for j in children:
            x, u = int(tokens[j]), float(uniforms[j])
            inside = 0 <= x < limit
            px, qx = (float(p[x]) if inside else 0.0), (1.0 if q is None else float(q[x]) if inside else 0.0)
            if px > u * qx:
                taken = j
                break
            if q is None:
                if inside:
                    p[x] = 0.0
            else:
                p = torch.clamp(p - q, min=0.0)
            p = p / p.sum() if float(p.sum()) > 0 else p * 0
        if taken is None:
            p = p if float(p.sum()) > 0 else whole
            sums = torch.cumsum(p, 0)
            over = ((sums > float(uniforms[0]) * float(sums[-1])) & (p > 0)).nonzero()
            return path, int(over[0]) if len(over) else int((p > 0).nonzero()[-1])
        node = taken
        path.append(node)


def compact(pool, table, past, paths):
    """pool [layers, pages, heads, 64, width] changed in place; paths: a list of nodes a sequence."""
    for s, path in enumerate(paths):
        p = int(past[s])
        rows = [pool[:, int(table[s, (p + j) // PAGE]), :, (p + j) % PAGE].clone() for j in path]
        for i, row in enumerate(rows):
            pool[:, int(table[s, (p + i) // PAGE]), :, (p + i) % PAGE] = row
