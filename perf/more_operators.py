"""The operators of drafted tokens, as cases to measure.

A program that drafts several tokens ahead (a small model, or a look into the text so far) and lets the large model judge
them all in one step needs, next to each other:

* ``tree``: from the parents of every sequence's drafted nodes, what each node sees of its step (itself and those it
  continues, as bits) and its position in the text;
* ``attention``: the step's nodes against the paged cache, a node seeing the rows before the step (all, or the last
  ``window`` positions) and of the step's own rows those that its bits name;
* ``verify``: which nodes the target's probabilities accept, from given random numbers, and the token behind the last of
  them. Node 0 of a sequence is its newest certain token. At an accepted node its drafted children are tried in their
  order: with p the target's distribution there and q the one that the children were drawn from, child x is accepted with
  probability min(1, p(x) / q(x)); after a refusal p becomes max(p - q, 0) over its sum. Drafts without probabilities are
  certain ones: q(x) = 1. Where no child is left the next token is drawn from what p has become;
* ``compact``: the rows of the accepted nodes move together behind the rows from before the step, in all layers.

``run`` without ``own`` computes them from elementary operations; with ``own`` it calls this library. ``exact`` is a
separate statement of the same definitions in 64 bits.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
PAGE = 64
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _tree(name, n, nodes, shape, window=0):
    """``nodes``: (least, most) of a sequence. ``shape``: how a node finds its parent (``_parents``)."""
    case = dict(kind="tree", n=n, nodes_lo=nodes[0], nodes_hi=nodes[1], shape=shape, window=window)
    return dict(name=name, **case) if name else case


def _attention(name, dtype, heads, kv_heads, dim, n, past, nodes, shape, window=0):
    case = dict(kind="attention", dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, n=n, past_lo=past[0], past_hi=past[1],
                nodes_lo=nodes[0], nodes_hi=nodes[1], shape=shape, window=window)
    return dict(name=name, **case) if name else case


def _verify(name, n, nodes, shape, vocab, limit, temperature, drawn, floors=False):
    """``drawn``: drafts were drawn from distributions that are at hand; else they are certain ones. ``floors``: only the
    largest logits of a row have probability."""
    case = dict(kind="verify", n=n, nodes_lo=nodes[0], nodes_hi=nodes[1], shape=shape, vocab=vocab, limit=limit, temperature=temperature,
                drawn=drawn, floors=floors)
    return dict(name=name, **case) if name else case


def _compact(name, dtype, layers, kv_heads, dim, n, past, nodes, kept):
    """``kept``: (least, most) nodes of a sequence that stay, the first one included."""
    case = dict(kind="compact", dtype=dtype, layers=layers, kv_heads=kv_heads, dim=dim, n=n, past_lo=past[0], past_hi=past[1],
                nodes_lo=nodes[0], nodes_hi=nodes[1], kept_lo=kept[0], kept_hi=kept[1])
    return dict(name=name, **case) if name else case


def listed():
    return [
        # One chat: a token and seven drafted behind it, two or three a level. All latency.
        _tree("tree-chat", 1, (8, 8), 3),
        # A full batch of unequal trees, the widest that are drafted.
        _tree("tree-batch64", 64, (17, 250), 0, window=4096),
        # One chat on a text of 2,000 tokens: five tokens in a row.
        _attention("chain-chat", "bf16", 16, 8, 128, 1, (2000, 2000), (5, 5), 1),
        # A busy server: 64 sequences of unequal length, eight nodes each.
        _attention("batch64", "bf16", 32, 8, 128, 64, (150, 4096), (8, 8), 2),
        # Few long texts, a broader tree.
        _attention("long-texts", "bf16", 32, 8, 128, 4, (9000, 30000), (11, 24), 4),
        # The broadest trees on ordinary texts: 256 rows of queries a key/value head, the most arithmetic.
        _attention("broad-trees", "bf16", 32, 8, 128, 8, (1000, 8192), (40, 64), 0),
        # The 32-bit path of a small model under a window, ragged.
        _attention("window-fp32", "fp32", 8, 4, 64, 5, (33, 700), (1, 13), 3, window=256),
        # One chat with a small model as its drafter.
        _verify("verify-chat", 1, (6, 6), 1, 151936, 151936, 0.8, True),
        # A full batch with a small model as its drafter: the most bytes.
        _verify("verify-batch64", 64, (3, 6), 1, 151936, 151669, 1.0, True),
        # Trees out of the texts so far, whose drafts have no probabilities.
        _verify("verify-trees", 8, (16, 24), 4, 151936, 151936, 0.7, False),
        # After the step of one chat, all layers.
        _compact("compact-chat", "bf16", 28, 8, 128, 1, (2000, 2000), (8, 8), (4, 4)),
        # After the step of a batch, all layers.
        _compact("compact-batch", "bf16", 28, 8, 128, 24, (60, 250), (8, 40), (1, 7)),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tree", "attention", "attention", "attention", "verify", "verify", "compact"])
    shape = rng.choice([0, 0, 1, 2, 3, 4, 7])
    if kind == "tree":
        nodes = _log_int(rng, 1, 256)
        return _tree("", _log_int(rng, 1, 64), (max(1, nodes // rng.choice([1, 2, 9])), nodes), shape, rng.choice([0, 0, _log_int(rng, 1, 3000)]))
    if kind == "verify":
        n, nodes = _log_int(rng, 1, 64), _log_int(rng, 1, 32)
        vocab = _log_int(rng, 300, 152000)
        nodes = max(1, min(nodes, 320 * 152000 // (n * vocab)))
        return _verify("", n, (max(1, nodes // rng.choice([1, 2, 5])), nodes), shape, vocab, max(1, vocab - rng.choice([0, 0, 1, 131])),
                       rng.choice([0.0, 0.3, 0.8, 1.0, 1.7]), rng.random() < 0.6, rng.random() < 0.3)
    dtype = rng.choice(["bf16"] * 4 + ["fp32"])
    if kind == "compact":
        layers, (kv_heads, dim) = rng.choice([1, 3, 28]), rng.choice([(8, 128), (8, 64), (4, 64), (3, 24)])
        n, nodes = _log_int(rng, 1, 24), _log_int(rng, 1, 64)
        past, kept = _log_int(rng, 1, max(2, min(2000, 5000 // n))), rng.randint(1, nodes)
        return _compact("", dtype, layers, kv_heads, dim, n, (past // 3, past), (max(1, nodes // rng.choice([1, 2])), nodes), (max(1, kept // 4), kept))
    heads, kv_heads, dim = rng.choice([(16, 8, 128), (32, 8, 128), (32, 8, 64), (8, 8, 64), (16, 2, 128), (40, 8, 128), (6, 3, 24)] if dtype == "bf16" else
                                      [(16, 8, 128), (8, 4, 64), (6, 3, 24), (4, 2, 16)])
    n = _log_int(rng, 1, 64 if dtype == "bf16" else 8)
    nodes = _log_int(rng, 1, max(1, min(256, 500 // n)))
    most = min(30000, 130000 // n, 500 * 6000 // (n * nodes)) if dtype == "bf16" and dim >= 64 else 3000 // n
    past = _log_int(rng, 4, max(5, most))
    window = 0 if rng.random() < 0.6 else _log_int(rng, 1, past + nodes)
    return _attention("", dtype, heads, kv_heads, dim, n, (rng.choice([0, past // 3, past]), past), (max(1, nodes // rng.choice([1, 2, 9])), nodes), shape, window)


# ------------------------------------------------------------------ inputs ----

def _spread(lo, hi, n, salt):
    """``n`` lengths from lo to hi, hi among them; they belong to the case, not to the seed."""
    rng = random.Random(f"{lo} {hi} {n} {salt}")
    out = [rng.randint(lo, hi) for _ in range(n)]
    out[rng.randrange(n)] = hi
    return out


def _counts(case):
    return _spread(case["nodes_lo"], case["nodes_hi"], case["n"], "nodes")


def _past(case):
    return _spread(case["past_lo"], case["past_hi"], case["n"], "past")


def _parents(case, counts, rng):
    """Per sequence the parent of each node, -1 for the first. Shape 0: any earlier node, near ones rather; 1: the node
    before; w > 1: levels of up to w nodes, each continuing some node of the level above."""
    out = []
    for count in counts:
        parents, level = [-1], [0]
        while len(parents) < count:
            if case["shape"] == 0:
                i = len(parents)
                parents.append(max(0, i - 1 - int(rng.expovariate(0.15))))
            elif case["shape"] == 1:
                parents.append(len(parents) - 1)
            else:
                i = len(parents)
                width = min(rng.randint(1, case["shape"]), count - i)
                parents += sorted(rng.choice(level) for _ in range(width))
                level = list(range(i, i + width))
        out.append(parents)
    return out


def _depths(parents):
    depth = []
    for p in parents:
        depth.append(0 if p < 0 else depth[p] + 1)
    return depth


def _ways(parents, depth, window, words):
    """The nodes that each node sees, as ``words`` 32-bit words a node: itself and those it continues, in the window."""
    out = np.zeros((len(parents), words), dtype=np.uint32)
    for i in range(len(parents)):
        j = i
        while j >= 0 and (window == 0 or depth[i] - depth[j] < window):
            out[i, j // 32] |= np.uint32(1 << (j % 32))
            j = parents[j]
    return out.view(np.int32)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def prepare(case, seed):
    """What a program holds before the call: the step's tables, the cache's pools with their block table (pages in no
    order), queries, logits, buffers for the results."""
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(int(seed))
    rng = random.Random(f"{case['kind']} {seed}")
    n, counts = case["n"], _counts(case)
    starts = [0]
    for c in counts:
        starts.append(starts[-1] + c)
    T, most = starts[-1], max(counts)
    s = dict(case=case, counts=_ints(counts), seq_start=_ints(starts), max_count=most)
    if case["kind"] != "compact":
        trees = _parents(case, counts, rng)
        s["parents"] = _ints([p for tree in trees for p in tree])
    if case["kind"] == "verify":
        return _prepare_verify(case, s, gen, T, n)
    words = -(-most // 32)
    if case["kind"] == "tree":
        s.update(past=_ints([rng.randint(0, 30000) for _ in range(n)]), seen=torch.zeros((T, words), dtype=torch.int32, device=DEVICE),
                 positions=torch.zeros(T, dtype=torch.int32, device=DEVICE))
        return s
    past, dtype, K, dim = _past(case), DTYPES[case["dtype"]], case["kv_heads"], case["dim"]
    longest = max(p + c for p, c in zip(past, counts))
    stride = -(-longest // PAGE)
    n_pages = n * stride + 3
    table = torch.randperm(n_pages, generator=gen, device=DEVICE)[:n * stride].to(torch.int32).view(n, stride).contiguous()
    s.update(past=_ints(past), table=table, longest=longest)
    if case["kind"] == "compact":
        s["pools"] = torch.randn((case["layers"], 2, n_pages, K, PAGE, dim), generator=gen, device=DEVICE, dtype=torch.float32 if dtype == torch.float32 else dtype)
        # a way through each tree: its first nodes may lie in place already, the others lie behind all places that are filled
        paths = np.full((n, most), -1, dtype=np.int32)
        kept = [min(c, k) for c, k in zip(counts, _spread(case["kept_lo"], case["kept_hi"], n, "kept"))]
        for i, (c, k) in enumerate(zip(counts, kept)):
            there = 1 + rng.randint(0, k - 1)
            while c - k < k - there:
                there += 1
            paths[i, :k] = list(range(there)) + sorted(rng.sample(range(k, c), k - there))
        s.update(path=torch.from_numpy(paths).to(DEVICE), lengths=_ints(kept))
        return s
    depths = [_depths(tree) for tree in trees]
    seen = np.concatenate([_ways(tree, depth, case["window"], words) for tree, depth in zip(trees, depths)])
    # queries twice as long as keys: some heads look at few rows, as trained ones do
    q = (2.0 * torch.randn((T, case["heads"], dim), generator=gen, device=DEVICE)).to(dtype)
    pools = [torch.randn((n_pages, K, PAGE, dim), generator=gen, device=DEVICE).to(dtype) for _ in range(2)]
    s.update(q=q, k_pool=pools[0], v_pool=pools[1], seen=torch.from_numpy(seen).to(DEVICE), scale=dim ** -0.5,
             positions=_ints([p + d for p, depth in zip(past, depths) for d in depth]), out=torch.empty((T, case["heads"] * dim), dtype=dtype, device=DEVICE))
    return s


def _prepare_verify(case, s, gen, T, n):
    vocab, limit, warm = case["vocab"], case["limit"], case["temperature"] or 1.0

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=DEVICE)

    # both models agree on most of it: a common part, sharp as logits of a language model are, and a difference
    common = 2.5 * normal(T, vocab)
    logits = common + 0.7 * normal(T, vocab)
    starts, parents = s["seq_start"].long(), s["parents"].long()
    base = torch.repeat_interleave(starts[:-1], s["counts"].long())
    above = torch.where(parents >= 0, base + parents, base + 0 * parents)
    if case["drawn"]:
        probs = torch.softmax((common + 0.7 * normal(T, vocab))[:, :limit] / warm, dim=1)
        probs = torch.nn.functional.pad(probs, (0, vocab - limit)).contiguous()
        tokens = torch.multinomial(probs, 64, replacement=True, generator=gen)
    else:
        probs = None
        tokens = torch.topk(logits[:, :limit], min(limit, 8), dim=1).indices
    del common
    # node t is one of its parent's draws; certain drafts are among the likeliest tokens
    pick = torch.randint(0, tokens.shape[1], (T,), generator=gen, device=DEVICE)
    s.update(logits=logits, probs=probs, tokens=tokens[above, pick].to(torch.int32), uniforms=torch.rand(T, generator=gen, device=DEVICE),
             path=torch.zeros((n, s["max_count"]), dtype=torch.int32, device=DEVICE), lengths=torch.zeros(n, dtype=torch.int32, device=DEVICE),
             chosen=torch.zeros(n, dtype=torch.int32, device=DEVICE), floors=None)
    if case["floors"]:
        s["floors"] = torch.topk(logits[:, :limit], min(limit, 50), dim=1).values[:, -1].contiguous()
    return s


# ------------------------------------------------------------------ one pass ----

def run(state):
    kind = state["case"]["kind"]
    return (_OWN if own else _PLAIN)[kind](state)


def _own_tree(s):
    from sleuth_b200.kernels import ops
    ops.draft_tree(s["parents"], s["seq_start"], s["past"], s["counts"], s["seen"], s["positions"], s["max_count"], s["case"]["window"])
    return {"seen": s["seen"], "positions": s["positions"]}


def _own_attention(s):
    from sleuth_b200.kernels import ops
    c = s["case"]
    if "scratch" not in s:      # a program's workspace, made once
        floats = ops.attention_tree_scratch_floats(s["q"].shape[0], c["n"], s["max_count"], c["heads"], c["kv_heads"], c["dim"], s["longest"], s["q"].dtype)
        s["scratch"] = torch.empty(floats, dtype=torch.float32, device=DEVICE) if floats else None
    ops.attention_tree(s["q"], s["k_pool"], s["v_pool"], s["out"], s["seq_start"], s["past"], s["counts"], s["seen"], s["positions"], s["table"],
                       s["max_count"], c["heads"], c["kv_heads"], c["dim"], c["window"], s["scale"], scratch=s["scratch"], max_keys=s["longest"])
    return {"out": s["out"]}


def _own_verify(s):
    from sleuth_b200.kernels import ops
    c = s["case"]
    if "scratch" not in s:
        words = ops.verify_drafts_scratch_words(c["n"], s["logits"].shape[0], c["limit"], drawn=c["drawn"])
        s["scratch"] = torch.empty(words, dtype=torch.int32, device=DEVICE) if words else None
    ops.verify_drafts(s["logits"], c["limit"], s["tokens"], s["parents"], s["seq_start"], s["counts"], s["uniforms"], c["temperature"], s["path"],
                      s["lengths"], s["chosen"], s["max_count"], probs=s["probs"], floors=s["floors"], scratch=s["scratch"])
    return {"path": s["path"], "lengths": s["lengths"], "chosen": s["chosen"]}


def _own_compact(s):
    from sleuth_b200.kernels import ops
    ops.cache_compact(s["pools"], s["table"], s["past"], s["path"], s["lengths"])
    return {"pools": s["pools"]}


def _plain_tree(s):
    """Who is whose parent as a 0/1 matrix a sequence; its powers say who is above whom, doubling the distance each time."""
    n, C, window = s["case"]["n"], s["max_count"], s["case"]["window"]
    node = torch.arange(C, device=DEVICE)
    at = (s["seq_start"][:n].long()[:, None] + node).clamp(max=s["parents"].numel() - 1)
    real = node < s["counts"].long()[:, None]
    parents = torch.where(real, s["parents"].long()[at], torch.full_like(at, -1))
    up = (parents[:, :, None] == node).float()
    way = torch.eye(C, device=DEVICE).expand(n, C, C)
    reach = 1
    while reach < C:
        way = ((way + torch.matmul(way, up)) > 0).float()
        up = torch.matmul(up, up)
        reach *= 2
    depth = way.sum(2).long() - 1
    if window:
        way = way * ((depth[:, :, None] - depth[:, None, :]) < window).float()
    words = s["seen"].shape[1]
    bits = torch.zeros((n, C, words * 32), dtype=torch.int64, device=DEVICE)
    bits[:, :, :C] = (way > 0) & real[:, :, None]
    packed = (bits.view(n, C, words, 32) << torch.arange(32, device=DEVICE)).sum(3)
    packed = torch.where(packed >= 1 << 31, packed - (1 << 32), packed).to(torch.int32)
    return {"seen": packed[real], "positions": (s["past"].long()[:, None] + depth)[real].to(torch.int32)}


def _plain_attention(s):
    c = s["case"]
    n, H, K, dim, C, L = c["n"], c["heads"], c["kv_heads"], c["dim"], s["max_count"], s["longest"]
    past, counts = s["past"].long(), s["counts"].long()

    def rows(pool):
        return pool[s["table"].long()].permute(0, 2, 1, 3, 4).reshape(n, K, -1, dim)[:, :, :L].float()

    node, key = torch.arange(C, device=DEVICE), torch.arange(L, device=DEVICE)
    token = (s["seq_start"][:n].long()[:, None] + node).clamp(max=s["q"].shape[0] - 1)                         # [n, C]
    q = s["q"].float()[token].view(n, C, K, H // K, dim).permute(0, 2, 3, 1, 4).reshape(n, K, (H // K) * C, dim)
    scores = (torch.matmul(q, rows(s["k_pool"]).transpose(2, 3)) * s["scale"]).view(n, K, H // K, C, L)
    new = key[None, :] - past[:, None]                                                                         # [n, L]: the key as a node of the step
    bits = torch.repeat_interleave(s["seen"].long()[token], 32, dim=2) >> (torch.arange(s["seen"].shape[1] * 32, device=DEVICE) % 32) & 1
    pick = new.clamp(0, bits.shape[2] - 1)[:, None, :].expand(n, C, L)
    sees = (bits.gather(2, pick) > 0) & (new >= 0)[:, None, :] & (new < counts[:, None])[:, None, :]
    old = (new < 0)[:, None, :].expand(n, C, L)
    if c["window"]:
        old = old & (key > s["positions"].long()[token][:, :, None] - c["window"])
    sees = ((sees | old) & (node < counts[:, None])[:, :, None])[:, None, None]
    scores = torch.where(sees, scores, torch.full_like(scores, -math.inf))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    held = (key < (past + counts)[:, None])[:, None, :, None]
    y = torch.matmul(p.view(n, K, (H // K) * C, L), torch.where(held, rows(s["v_pool"]), torch.zeros((), device=DEVICE)))
    y = y.view(n, K, H // K, C, dim).permute(0, 3, 1, 2, 4).reshape(n, C, H * dim)
    return {"out": y[node < counts[:, None]].to(s["q"].dtype)}


def _weights_of(logits, floors, temperature):
    """64-bit probabilities of rows of logits: nothing below the floor; all of it on the first largest at temperature 0."""
    x = logits.double()
    if temperature <= 0:
        return torch.nn.functional.one_hot(x.argmax(-1), x.shape[-1]).double()
    x = x / temperature
    e = torch.exp(x - x.amax(-1, keepdim=True))
    if floors is not None:
        e = torch.where(logits >= floors[:, None], e, torch.zeros_like(e))
    return e / e.sum(-1, keepdim=True)


def _plain_verify(s):
    """One sweep over the nodes in their order, all sequences at once: a node is tried if it continues the one reached."""
    c = s["case"]
    n, limit, greedy = c["n"], c["limit"], c["temperature"] <= 0
    first, counts = s["seq_start"][:n].long(), s["counts"].long()
    reached = torch.zeros(n, dtype=torch.long, device=DEVICE)
    length = torch.ones(n, dtype=torch.long, device=DEVICE)
    path = torch.full((n, s["max_count"] + 1), -1, dtype=torch.long, device=DEVICE)
    path[:, 0] = 0
    every = torch.arange(n, device=DEVICE)

    def row(t):
        return _weights_of(s["logits"][t, :limit], None if s["floors"] is None else s["floors"][t], c["temperature"])

    left = row(first)                                # what p has become at the node reached, in all 1
    for j in range(1, s["max_count"]):
        t = (first + j).clamp(max=s["parents"].numel() - 1)
        tried = (j < counts) & (s["parents"].long()[t] == reached)
        x = s["tokens"].long()[t]
        inside = x < limit
        at = x.clamp(max=limit - 1)
        p = torch.where(inside, left[every, at], torch.zeros_like(left[:, 0]))
        if s["probs"] is not None and not greedy:
            q_row = s["probs"][first + reached, :limit].double()
            q = torch.where(inside, q_row[every, at], torch.zeros_like(p))
        else:
            q_row, q = None, torch.ones_like(p)
        taken = tried & (p > s["uniforms"][t].double() * q) if not greedy else tried & (p > 0)
        refused = tried & ~taken
        if q_row is None:
            rest = torch.where(inside[:, None] & (torch.arange(limit, device=DEVICE) == at[:, None]), torch.zeros_like(left), left)
        else:
            rest = (left - q_row).clamp(min=0)
        if not greedy:
            left = torch.where(refused[:, None], rest / rest.sum(1, keepdim=True).clamp(min=1e-300), left)
        reached = torch.where(taken, torch.full_like(reached, j), reached)
        path.scatter_(1, torch.where(taken, length, torch.full_like(length, s["max_count"]))[:, None], torch.full((n, 1), j, device=DEVICE))
        length = length + taken
        left = torch.where(taken[:, None], row(first + reached), left)
    path[:, s["max_count"]] = -1
    sums = left.cumsum(1)
    chosen = (sums <= s["uniforms"][first].double()[:, None] * sums[:, -1:]).sum(1) if not greedy else left.argmax(1)
    return {"path": path[:, :-1].to(torch.int32), "lengths": length.to(torch.int32), "chosen": chosen.clamp(max=limit - 1).to(torch.int32)}


def _plain_compact(s):
    c = s["case"]
    place = torch.arange(s["path"].shape[1], device=DEVICE)
    moves = (place < s["lengths"][:, None]) & (s["path"] != place)
    table, K, past = s["table"].long(), c["kv_heads"], s["past"].long()[:, None]
    seq = torch.arange(c["n"], device=DEVICE)[:, None]

    def rows(i):      # of a layer's keys or values, all heads: [moves, K]
        i = torch.where(moves, past + i, past)
        i = torch.where(moves, i, torch.zeros_like(i))
        return ((table[seq, i // PAGE][..., None] * K + torch.arange(K, device=DEVICE)) * PAGE + (i % PAGE)[..., None]).reshape(-1)

    to, of = rows(place), rows(s["path"].long())
    flat = s["pools"].view(c["layers"] * 2, -1, c["dim"])
    flat[:, to] = flat[:, of]
    return {"pools": s["pools"]}


_OWN = dict(tree=_own_tree, attention=_own_attention, verify=_own_verify, compact=_own_compact)
_PLAIN = dict(tree=_plain_tree, attention=_plain_attention, verify=_plain_verify, compact=_plain_compact)


# ------------------------------------------------------------------ what a pass cannot do without ----

def work(case):
    counts = _counts(case)
    T, most, n = sum(counts), max(counts), case["n"]
    if case["kind"] == "tree":
        return {"bytes": 4 * T * (2 + -(-most // 32)) + 12 * n, "flops": 0}
    if case["kind"] == "verify":
        # the rows of one way from the first node down, and q once where a draft is refused
        levels = [c if case["shape"] == 1 else 1 + math.ceil(math.log2(c)) if case["shape"] == 0 else 1 + math.ceil(2 * (c - 1) / (1 + case["shape"])) for c in counts]
        rows = sum(levels) + (n if case["drawn"] and case["temperature"] > 0 else 0)
        return {"bytes": 4 * rows * case["limit"] + 16 * T + 4 * n * (2 + most), "flops": 0}
    size, K, dim = (2 if case["dtype"] == "bf16" else 4), case["kv_heads"], case["dim"]
    if case["kind"] == "compact":
        kept = [min(c, k) for c, k in zip(counts, _spread(case["kept_lo"], case["kept_hi"], n, "kept"))]
        return {"bytes": 2 * sum(k / 2 for k in kept) * case["layers"] * 2 * K * dim * size, "flops": 0}
    H, rows, pairs = case["heads"], 0, 0
    for p, c in zip(_past(case), counts):
        deep = min(p, case["window"]) if case["window"] else p
        rows += deep + c
        pairs += (deep + 1 + math.log2(c)) * c
    return {"bytes": rows * K * 2 * dim * size + T * (H * 2 * dim * size + 4 * -(-most // 32)), "flops": 4 * pairs * H * dim}


# ------------------------------------------------------------------ 64 bits ----

def exact(case, seed):
    s = prepare(case, seed)
    return dict(tree=_exact_tree, attention=_exact_attention, verify=_exact_verify, compact=_exact_compact)[case["kind"]](s)


def _exact_tree(s):
    case, counts, parents, at = s["case"], _counts(s["case"]), s["parents"].tolist(), 0
    seen, positions = [], []
    for c, p in zip(counts, s["past"].tolist()):
        tree = parents[at:at + c]
        depth = _depths(tree)
        seen.append(_ways(tree, depth, case["window"], s["seen"].shape[1]))
        positions += [p + d for d in depth]
        at += c
    return {"seen": torch.from_numpy(np.concatenate(seen)), "positions": torch.tensor(positions, dtype=torch.int32)}


def _exact_attention(s):
    case = s["case"]
    K, G, dim = case["kv_heads"], case["heads"] // case["kv_heads"], case["dim"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEVICE)
    seen, start = s["seen"].cpu().numpy().view(np.uint32), 0
    for i, (p, c) in enumerate(zip(_past(case), _counts(case))):
        end = p + c
        pages = s["table"][i, :-(-end // PAGE)].long()
        dark = torch.zeros((c, end), dtype=torch.bool, device=DEVICE)
        dark[:, p:] = torch.tensor([[not int(seen[start + a, b // 32]) >> (b % 32) & 1 for b in range(c)] for a in range(c)], device=DEVICE)
        if case["window"]:
            dark[:, :p] = torch.arange(p, device=DEVICE) <= s["positions"][start:start + c].long()[:, None] - case["window"]
        for k in range(K):
            keys = s["k_pool"][pages, k].reshape(-1, dim)[:end].double()
            values = s["v_pool"][pages, k].reshape(-1, dim)[:end].double()
            a = torch.einsum("chd,kd->hck", s["q"][start:start + c, k * G:(k + 1) * G].double(), keys) * s["scale"]
            a = torch.softmax(a.masked_fill_(dark, -math.inf), dim=2)
            out[start:start + c, k * G * dim:(k + 1) * G * dim] = torch.einsum("hck,kd->chd", a, values).reshape(c, G * dim)
        start += c
    return {"out": out}


def _exact_verify(s):
    """A sequence at a time, as the definition reads."""
    case, limit, n = s["case"], s["case"]["limit"], s["case"]["n"]
    tokens, parents, uniforms = s["tokens"].tolist(), s["parents"].tolist(), s["uniforms"].double().tolist()
    path, lengths, chosen = np.full((n, s["max_count"]), -1, dtype=np.int32), [], []
    start = 0
    for i, count in enumerate(_counts(case)):
        node, way = 0, [0]
        while True:
            logits = s["logits"][start + node, :limit].double()
            if case["temperature"] <= 0:
                best = int(torch.nonzero(logits == logits.max())[0])
                nxt = [j for j in range(node + 1, count) if parents[start + j] == node and tokens[start + j] == best]
                if not nxt:
                    chosen.append(best)
                    break
                node = nxt[0]
                way.append(node)
                continue
            keep = torch.ones(limit, dtype=torch.bool, device=DEVICE) if s["floors"] is None else s["logits"][start + node, :limit] >= s["floors"][start + node]
            p = torch.softmax((logits / case["temperature"]).masked_fill(~keep, -math.inf), dim=0)
            q = None if s["probs"] is None else s["probs"][start + node, :limit].double()
            taken = None
            for j in range(node + 1, count):
                if parents[start + j] != node:
                    continue
                x = tokens[start + j]
                px, qx = (float(p[x]) if x < limit else 0.0), (1.0 if q is None else float(q[x]) if x < limit else 0.0)
                if px > uniforms[start + j] * qx:
                    taken = j
                    break
                if q is None:
                    if x < limit:
                        p[x] = 0.0
                else:
                    p = torch.clamp(p - q, min=0.0)
                p = p / p.sum()
            if taken is None:
                c = torch.cumsum(p, 0)
                chosen.append(min(int(torch.searchsorted(c, uniforms[start] * float(c[-1]), right=True)), limit - 1))
                break
            node = taken
            way.append(node)
        path[i, :len(way)] = way
        lengths.append(len(way))
        start += count
    return {"path": torch.from_numpy(path), "lengths": torch.tensor(lengths, dtype=torch.int32), "chosen": torch.tensor(chosen, dtype=torch.int32)}


def _exact_compact(s):
    """Row by row, on the host's word."""
    pools, table, path = s["pools"], s["table"].tolist(), s["path"].tolist()
    for i, (p, length) in enumerate(zip(_past(s["case"]), s["lengths"].tolist())):
        rows = [(p + j, p + path[i][j]) for j in range(length)]
        held = [pools[:, :, table[i][b // PAGE], :, b % PAGE].clone() for _, b in rows]
        for (a, _), row in zip(rows, held):
            pools[:, :, table[i][a // PAGE], :, a % PAGE] = row
    return {"pools": pools}
