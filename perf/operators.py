"""The operators of a cache of bounded size, as cases to measure.

A program that serves texts longer than it can hold keeps, for every sequence, the first few tokens, the latest ones and
those that queries have looked at most. Three things are needed for that, next to each other:

* ``attention``: the new tokens of a step (a prompt, a portion of one, a few tokens or one) against the paged cache,
  where a query sees the last ``window`` rows and the first ``first`` ones;
* the same with ``weights``: the step's softmax weights, summed over the step's queries and over the query heads of a
  key/value head, join what every cache row has gathered so far;
* ``evict``: of the rows that a sequence holds, ``budget`` stay: its first positions, its latest ones and those with the
  largest gathered weight; the rows that stay but lie behind the budget move into the places of those that go.

``run`` without ``own`` computes them from elementary operations in 32 bits; with ``own`` it calls this library.
``exact`` is a separate statement of the same definitions in 64 bits.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda:0"
PAGE = 64
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _attention(name, dtype, heads, kv_heads, dim, n, past, count, window=0, first=0, weights=False):
    """``past`` and ``count``: (least, most) rows in the cache before the step and new tokens of a sequence."""
    case = dict(kind="attention", dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, n=n, past_lo=past[0], past_hi=past[1],
                count_lo=count[0], count_hi=count[1], window=window, first=first, weights=weights)
    return dict(name=name, **case) if name else case


def _evict(name, dtype, kv_heads, dim, n, length, past_rows, budget, first, recent, gone):
    """``length``: (least, most) rows that a sequence holds; ``past_rows``: whether all but the last of them were there
    before the step (else none was); ``gone``: how many tokens were evicted before."""
    case = dict(kind="evict", dtype=dtype, kv_heads=kv_heads, dim=dim, n=n, len_lo=length[0], len_hi=length[1], past_rows=past_rows,
                budget=budget, first=first, recent=recent, gone=gone)
    return dict(name=name, **case) if name else case


def listed():
    return [
        # One chat that has been going on for long: a token, of which the first four rows and the last 1,024 are seen.
        _attention("token-stream", "bf16", 16, 8, 128, 1, (5200, 5200), (1, 1), window=1024, first=4),
        # A busy server with a window: 64 sequences of unequal length, some shorter than the window.
        _attention("token-batch64", "bf16", 32, 8, 128, 64, (150, 4096), (1, 1), window=2048, first=64),
        # Eight sequences at a budget of 2,048 rows: every token's weights are gathered for the eviction that follows.
        _attention("token-weights8", "bf16", 16, 8, 128, 8, (2048, 2048), (1, 1), weights=True),
        # Few long texts before anything was evicted: the cache is what there is to read.
        _attention("token-weights-long", "bf16", 32, 8, 128, 6, (9000, 30000), (1, 1), weights=True),
        # The 32-bit path, small heads, a batch that goes on token by token.
        _attention("token-fp32", "fp32", 8, 4, 64, 5, (33, 700), (1, 1), window=256, first=4, weights=True),
        # A few tokens at a time (a user's short turn) on a bounded cache.
        _attention("turn-weights", "bf16", 32, 8, 128, 4, (1024, 2048), (3, 13), weights=True),
        # One prompt under a window: the work grows with the length times the window.
        _attention("prompt-window", "bf16", 16, 8, 128, 1, (0, 0), (2048, 2048), window=512, first=16),
        # Portions of long prompts on what the cache holds, unequal on both sides.
        _attention("portion-ragged", "bf16", 32, 8, 64, 7, (0, 3000), (64, 1500), window=1000, first=100),
        # A whole long prompt whose weights are gathered: the largest of all.
        _attention("prompt-weights", "bf16", 32, 8, 128, 1, (0, 0), (6000, 6000), weights=True),
        # A test-sized model in 32 bits: odd sizes throughout.
        _attention("prompt-tiny-fp32", "fp32", 6, 3, 24, 4, (0, 9), (1, 40), window=11, first=3, weights=True),
        # Every token of a full batch pushes one row out of each key/value head's cache.
        _evict("evict-step", "bf16", 8, 128, 64, (2049, 2049), True, 2048, 4, 512, 7000),
        # After long prompts: a few thousand rows become a thousand.
        _evict("evict-prompts", "bf16", 8, 128, 8, (2500, 8192), False, 1024, 4, 256, 0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["bf16"] * 4 + ["fp32"])
    heads, kv_heads, dim = rng.choice([(16, 8, 128), (32, 8, 128), (32, 8, 64), (8, 8, 64), (16, 2, 128)] if dtype == "bf16" else
                                      [(16, 8, 128), (8, 4, 64), (6, 3, 24), (4, 2, 16)])
    kind = rng.choice(["token", "token", "turn", "prompt", "prompt", "evict", "evict"])
    most = 30000 if dtype == "bf16" else 3000
    if kind == "evict":
        n = _log_int(rng, 1, 64)
        hi = _log_int(rng, 40, min(20000, 131072 // n))
        step = rng.random() < 0.5
        budget = hi - 1 if step else max(8, _log_int(rng, 8, hi))
        first = rng.choice([0, 1, 4, 17])
        first = min(first, budget // 4)
        recent = rng.randint(0, budget - first) if rng.random() < 0.3 else budget // rng.choice([2, 4, 8])
        lo = hi if step else max(1, hi // rng.choice([1, 2, 5]))
        return _evict("", dtype, kv_heads, dim, n, (lo, hi), step, budget, first, min(recent, budget - first), _log_int(rng, 1, 9000) if step else 0)
    if kind == "token":
        n = _log_int(rng, 1, 64 if dtype == "bf16" else 8)
        hi = _log_int(rng, 8, min(most, 180000 // n))
        past, count = (max(0, hi // rng.choice([1, 2, 9])), hi), (1, 1)
    elif kind == "turn":
        n = _log_int(rng, 1, 8)
        hi = _log_int(rng, 8, min(most, 24000 // n))
        c = _log_int(rng, 2, 24)
        past, count = (hi // rng.choice([1, 3]), hi), (max(1, c // rng.choice([1, 4])), c)
    else:
        n = _log_int(rng, 1, 8)
        c = _log_int(rng, 24, (6000 if dtype == "bf16" else 700) // n)
        hi = rng.choice([0, 0, _log_int(rng, 1, 8000 // n)])
        if (c + hi) * c * n * heads > 6000 * 6000 * 32:
            hi = 0
        past, count = (hi // 3, hi), (max(1, c // rng.choice([1, 1, 3])), c)
    form = rng.randrange(3)
    window = 0 if form == 0 else _log_int(rng, 1, max(2, past[1] + count[1]))
    first = 0 if window == 0 else rng.choice([0, 1, 4, 64, 100])
    return _attention("", dtype, heads, kv_heads, dim, n, past, count, window, first, weights=form == 0 or rng.random() < 0.5)


# ------------------------------------------------------------------ inputs ----

def _spread(lo, hi, n, salt):
    """``n`` lengths from lo to hi, both among them where there is room; they belong to the case, not to the seed."""
    rng = random.Random(f"{lo} {hi} {n} {salt}")
    out = [rng.randint(lo, hi) for _ in range(n)]
    out[rng.randrange(n)] = hi
    return out


def _lengths(case):
    """Per sequence the rows before the step and the new ones."""
    if case["kind"] == "evict":
        lens = _spread(case["len_lo"], case["len_hi"], case["n"], "rows")
        past = [max(0, n - 1) if case["past_rows"] else 0 for n in lens]
        return past, [n - p for n, p in zip(lens, past)]
    return _spread(case["past_lo"], case["past_hi"], case["n"], "past"), _spread(case["count_lo"], case["count_hi"], case["n"], "count")


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def prepare(case, seed):
    """What a serving program holds before the call: the cache's pools with their block table (pages in no order), the
    step's tables, the queries, what the rows have gathered, buffers for the results."""
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(int(seed))
    dtype, n, K, dim = DTYPES[case["dtype"]], case["n"], case["kv_heads"], case["dim"]
    past, counts = _lengths(case)
    longest = max(p + c for p, c in zip(past, counts))
    stride = -(-longest // PAGE)
    n_pages = n * stride + 3
    pools = [torch.randn((n_pages, K, PAGE, dim), generator=gen, device=DEVICE).to(dtype) for _ in range(2)]
    table = torch.randperm(n_pages, generator=gen, device=DEVICE)[:n * stride].to(torch.int32).view(n, stride).contiguous()
    s = dict(case=case, k_pool=pools[0], v_pool=pools[1], table=table, past=_ints(past), counts=_ints(counts), longest=longest)
    cap = stride * PAGE
    # what rows gather spreads over orders of magnitude, and many have gathered nothing at all
    gathered = torch.exp(1.7 * torch.randn((n, K, cap), generator=gen, device=DEVICE)) * 0.05
    gathered = torch.where(torch.rand((n, K, cap), generator=gen, device=DEVICE) < 0.03, torch.zeros_like(gathered), gathered)
    if case["kind"] == "evict":
        # the positions of the rows that were there: the first tokens, the latest, and some in between, in no order
        lens = [p + c for p, c in zip(past, counts)]
        held = case["past_rows"]
        seen = [m + (case["gone"] if held else 0) for m in lens]
        places = torch.arange(cap, device=DEVICE).expand(n, K, cap)
        p, first, tail = s["past"].view(n, 1, 1), case["first"], (s["past"].view(n, 1, 1) + case["first"]) // 2
        at = torch.where(places < torch.minimum(p, torch.maximum(tail, torch.full_like(p, first))), places, places + (case["gone"] if held else 0))
        order = torch.where(places < p, torch.rand((n, K, cap), generator=gen, device=DEVICE), 2.0 + places).argsort(dim=-1)
        s.update(weights=gathered, positions=at.gather(-1, order).to(torch.int32).contiguous(), lengths=_ints(lens), seen=_ints(seen),
                 weights_out=torch.zeros_like(gathered), positions_out=torch.zeros((n, K, cap), dtype=torch.int32, device=DEVICE))
        return s
    H, T = case["heads"], sum(counts)
    starts = [0]
    for c in counts:
        starts.append(starts[-1] + c)
    # queries twice as long as keys: some heads look at few rows, as trained ones do
    q = (2.0 * torch.randn((T, H, dim), generator=gen, device=DEVICE)).to(dtype)
    seq_of = torch.repeat_interleave(torch.arange(n, device=DEVICE), s["counts"].long())
    index = torch.arange(T, device=DEVICE) - torch.tensor(starts[:-1], device=DEVICE)[seq_of]
    s.update(q=q, seq_start=_ints(starts), out=torch.empty((T, H * dim), dtype=dtype, device=DEVICE), seq_of=seq_of, index=index,
             max_count=max(counts), scale=dim ** -0.5)
    if case["weights"]:
        s.update(weights=gathered, weights_out=torch.zeros_like(gathered))
    return s


# ------------------------------------------------------------------ one pass ----

def run(state):
    if state["case"]["kind"] == "evict":
        return (_own_evict if own else _plain_evict)(state)
    return (_own_attention if own else _plain_attention)(state)


def _own_attention(s):
    from sleuth_b200.kernels import ops
    c = s["case"]
    if "scratch" not in s:      # a program's workspace, made once
        floats = ops.attention_kept_scratch_floats(s["q"].shape[0], c["n"], s["max_count"], c["heads"], c["kv_heads"], c["dim"], s["longest"],
                                                   s["q"].dtype, weights=c["weights"])
        s["scratch"] = torch.empty(floats, dtype=torch.float32, device=DEVICE) if floats else None
    ops.attention_kept(s["q"], s["k_pool"], s["v_pool"], s["out"], s["seq_start"], s["past"], s["counts"], s["table"], s["max_count"], c["heads"],
                       c["kv_heads"], c["dim"], c["window"], c["first"], s["scale"], scratch=s["scratch"], max_keys=s["longest"],
                       weights=s.get("weights"), weights_out=s.get("weights_out"))
    return {"out": s["out"], "weights": s["weights_out"]} if c["weights"] else {"out": s["out"]}


def _own_evict(s):
    from sleuth_b200.kernels import ops
    c = s["case"]
    if "scratch" not in s:
        words = ops.cache_evict_scratch_words(c["n"], c["kv_heads"], c["budget"], s["longest"])
        s["scratch"] = torch.empty(words, dtype=torch.int32, device=DEVICE) if words else None
    ops.cache_evict(s["weights"], s["positions"], s["k_pool"], s["v_pool"], s["table"], s["past"], s["lengths"], s["seen"], c["budget"], c["first"],
                    c["recent"], weights_out=s["weights_out"], positions_out=s["positions_out"], scratch=s["scratch"], max_length=s["longest"])
    return {"weights": s["weights_out"], "positions": s["positions_out"], "keys": s["k_pool"], "values": s["v_pool"]}


def _rows(pool, table):
    """The rows of every sequence in the order of the cache: [n, kv heads, rows, dim]."""
    n, stride = table.shape
    return pool[table.long()].permute(0, 2, 1, 3, 4).reshape(n, pool.shape[1], stride * PAGE, pool.shape[3])


def _plain_attention(s):
    c = s["case"]
    n, H, K, dim, C = c["n"], c["heads"], c["kv_heads"], c["dim"], s["max_count"]
    L = s["longest"]
    past, counts = s["past"].long(), s["counts"].long()
    keys, values = (_rows(p, s["table"])[:, :, :L].float() for p in (s["k_pool"], s["v_pool"]))
    slots = torch.arange(C, device=DEVICE)
    token = (s["seq_start"][:n].long()[:, None] + slots).clamp(max=s["q"].shape[0] - 1)                        # [n, C]
    q = s["q"].float()[token].view(n, C, K, H // K, dim).permute(0, 2, 3, 1, 4).reshape(n, K, (H // K) * C, dim)
    scores = (torch.matmul(q, keys.transpose(2, 3)) * s["scale"]).view(n, K, H // K, C, L)
    at, key = (past[:, None] + slots)[:, :, None], torch.arange(L, device=DEVICE)[None, None, :]
    seen = (key <= at) & (slots < counts[:, None])[:, :, None]
    if c["window"]:
        seen = seen & ((key > at - c["window"]) | (key < c["first"]))
    seen = seen[:, None, None]
    scores = torch.where(seen, scores, torch.full_like(scores, -math.inf))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    held = (torch.arange(L, device=DEVICE) < (past + counts)[:, None])[:, None, :, None]
    y = torch.matmul(p.view(n, K, (H // K) * C, L), torch.where(held, values, torch.zeros_like(values)))
    y = y.view(n, K, H // K, C, dim).permute(0, 3, 1, 2, 4).reshape(n, C, H * dim)
    out = y[s["seq_of"], s["index"]].to(s["q"].dtype)
    if not c["weights"]:
        return {"out": out}
    gained = p.sum((2, 3))                                                                                     # [n, K, L]
    before = torch.where(torch.arange(L, device=DEVICE) < past[:, None, None], s["weights"][:, :, :L], torch.zeros_like(gained))
    gathered = torch.zeros_like(s["weights"])
    gathered[:, :, :L] = torch.where(held[..., 0], before + gained, torch.zeros_like(gained))
    return {"out": out, "weights": gathered}


def _plain_evict(s):
    c = s["case"]
    n, K = c["n"], c["kv_heads"]
    w, cap = s["weights"], s["weights"].shape[2]
    place = torch.arange(cap, device=DEVICE)
    past, lens, seen = (s[k].long().view(n, 1, 1) for k in ("past", "lengths", "seen"))
    held = place < lens
    at = torch.where(place < past, s["positions"].long(), seen - lens + place)
    safe = (at < c["first"]) | (at >= seen - c["recent"])
    order = torch.where(held, torch.where(safe, torch.full_like(w, math.inf), w), torch.full_like(w, -math.inf))
    rank = torch.empty((n, K, cap), dtype=torch.long, device=DEVICE)
    rank.scatter_(2, torch.sort(order, dim=2, descending=True, stable=True).indices, place.expand(n, K, cap).contiguous())
    stays = held & (rank < c["budget"])
    left = torch.minimum(lens, torch.full_like(lens, c["budget"]))
    movers = torch.sort((~(stays & (place >= left))).to(torch.int32), dim=2, stable=True).indices              # rows to move, ascending, first
    hole = ((~stays) & (place < left)).long()
    nth = (hole.cumsum(2) - hole).clamp(min=0)
    source = torch.where(hole > 0, movers.gather(2, nth), place.expand(n, K, cap))
    source = torch.where(place < left, source, source[:, :, :1])
    filled = place < left
    weights = torch.where(filled, w.gather(2, source), torch.zeros_like(w))
    positions = torch.where(filled, at.gather(2, source), torch.zeros_like(source)).to(torch.int32)
    table, kv = s["table"].long(), torch.arange(K, device=DEVICE).view(1, K, 1)
    seq = torch.arange(n, device=DEVICE).view(n, 1, 1)

    def row_of(i):
        return (table[seq, i // PAGE] * K + kv) * PAGE + i % PAGE

    to = row_of(torch.where(place < left, place, torch.zeros_like(source))).reshape(-1)
    source = row_of(source).reshape(-1)
    for pool in (s["k_pool"], s["v_pool"]):
        flat = pool.view(-1, c["dim"])
        flat[to] = flat[source]
    return {"weights": weights, "positions": positions, "keys": s["k_pool"], "values": s["v_pool"]}


# ------------------------------------------------------------------ what a pass cannot do without ----

def _visible(case, past, count):
    """Pairs of query and key of one head, and rows that some query of the sequence sees."""
    w, f = case["window"], case["first"]
    pairs, rows = 0, 0
    for i in range(count):
        p = past + i
        if not w or w > p:
            pairs += p + 1
        else:
            pairs += w + min(f, p + 1 - w)
    end = past + count
    rows = end if not w else end - max(0, past + 1 - w) + min(f, max(0, past + 1 - w))
    return pairs, rows


def work(case):
    past, counts = _lengths(case)
    size, K, dim = (2 if case["dtype"] == "bf16" else 4), case["kv_heads"], case["dim"]
    if case["kind"] == "evict":
        size_of, total = 2 * dim * size, 0
        for p, c in zip(past, counts):
            n, b = p + c, case["budget"]
            total += K * (4 * n + 4 * p + 8 * min(n, b))
            if n > b:
                # rows that stay and lie behind the budget: the latest, and their share of the others that stay
                late = min(n - b, c if case["past_rows"] else case["recent"])
                others = max(0, n - case["first"] - case["recent"])
                behind = max(0, n - b - late)
                moves = late + (b - case["first"] - case["recent"]) * behind / max(1, others)
                total += K * 2 * size_of * moves
        return {"bytes": total, "flops": 0}
    H, pairs, rows, gathered = case["heads"], 0, 0, 0
    for p, c in zip(past, counts):
        a, b = _visible(case, p, c)
        pairs, rows, gathered = pairs + a, rows + b, gathered + 2 * p + c
    tokens = sum(counts)
    moved = rows * K * 2 * dim * size + tokens * H * 2 * dim * size + (4 * K * gathered if case["weights"] else 0)
    return {"bytes": moved, "flops": 4 * pairs * H * dim}


# ------------------------------------------------------------------ 64 bits ----

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "evict":
        return _exact_evict(s)
    past, counts = _lengths(case)
    K, G, dim = case["kv_heads"], case["heads"] // case["kv_heads"], case["dim"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEVICE)
    gathered = torch.zeros(s["weights"].shape, dtype=torch.float64, device=DEVICE) if case["weights"] else None
    start = 0
    for i, (p, c) in enumerate(zip(past, counts)):
        end = p + c
        pages = s["table"][i, :-(-end // PAGE)].long()
        at = torch.arange(p, end, device=DEVICE)
        key = torch.arange(end, device=DEVICE)
        dark = key[None, :] > at[:, None]
        if case["window"]:
            dark |= (key[None, :] <= at[:, None] - case["window"]) & (key[None, :] >= case["first"])
        for k in range(K):
            keys = s["k_pool"][pages, k].reshape(-1, dim)[:end].double()
            values = s["v_pool"][pages, k].reshape(-1, dim)[:end].double()
            gained = torch.zeros(end, dtype=torch.float64, device=DEVICE)
            for h in range(k * G, (k + 1) * G):
                a = s["q"][start:start + c, h].double() @ keys.T * s["scale"]
                a = torch.softmax(a.masked_fill_(dark, -math.inf), dim=1)
                out[start:start + c, h * dim:(h + 1) * dim] = a @ values
                gained += a.sum(0)
            if gathered is not None:
                gained[:p] += s["weights"][i, k, :p].double()
                gathered[i, k, :end] = gained
        start += c
    return {"out": out, "weights": gathered} if case["weights"] else {"out": out}


def _exact_evict(s):
    """On the host, a sequence and a key/value head at a time, as the definition reads."""
    c, (past, counts) = s["case"], _lengths(s["case"])
    weights, positions = s["weights"].double().cpu().numpy(), s["positions"].cpu().numpy()
    table = s["table"].cpu().numpy()
    pools = [s["k_pool"].cpu(), s["v_pool"].cpu()]
    new_w, new_p = weights * 0.0, positions * 0
    seen = s["seen"].cpu().numpy()
    for i, (p, n) in enumerate(zip(past, counts)):
        n += p
        left = min(n, c["budget"])
        for k in range(c["kv_heads"]):
            w = weights[i, k, :n]
            at = [int(positions[i, k, j]) if j < p else int(seen[i]) - n + j for j in range(n)]
            safe = [a < c["first"] or a >= seen[i] - c["recent"] for a in at]
            chosen = sorted(range(n), key=lambda j: (not safe[j], -w[j], j))[:left]
            stays = set(chosen)
            moves = dict(zip([d for d in range(left) if d not in stays], sorted(j for j in chosen if j >= left)))
            for d in range(left):
                j = moves.get(d, d)
                new_w[i, k, d], new_p[i, k, d] = w[j], at[j]
            if moves:
                to, of = (torch.tensor(v) for v in (list(moves.keys()), list(moves.values())))
                pages = torch.from_numpy(table[i]).long()
                for pool in pools:
                    pool[pages[to // PAGE], k, to % PAGE] = pool[pages[of // PAGE], k, of % PAGE]
    return {"weights": torch.from_numpy(new_w), "positions": torch.from_numpy(new_p), "keys": pools[0], "values": pools[1]}
