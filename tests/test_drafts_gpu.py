"""Drafted tokens: tree tables, attention over a tree, verification, compaction, and a run of them together, against the definitions in 64 bits."""

import math
import random

import pytest
import torch

from plain import drafts_plain as plain

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def make_tree(kind, count, rng):
    if kind == "chain":
        return [i - 1 for i in range(count)]
    if kind == "star":
        return [-1] + [0] * (count - 1) if count else []
    if kind == "forest":
        return [rng.choice([-1, *range(max(0, i - 4), i)]) for i in range(count)]
    return [-1 if i == 0 else max(0, i - 1 - int(rng.expovariate(0.4))) for i in range(count)]


def starts_of(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


# ------------------------------------------------------------------ tree tables ----

@pytest.mark.parametrize("window", [0, 1, 2, 7, 33, 64, 255, 256, 100000])
@pytest.mark.parametrize("kind", ["chain", "star", "random", "forest"])
@pytest.mark.parametrize("counts", [[1], [0], [8, 0, 1, 32], [33, 64, 2], [65, 128], [129, 256, 255, 3]])
def test_tree_tables(counts, kind, window):
    from sleuth_b200.kernels import ops
    rng = random.Random(f"{counts} {kind} {window}")
    trees = [make_tree(kind, c, rng) for c in counts]
    if kind == "forest" and counts[0] > 2:
        trees[0][1], trees[0][2] = 5, 2        # later nodes and itself are no parents
    most = max(1, max(counts))
    words = -(-most // 32) + (1 if window == 7 else 0)
    T, past = sum(counts), [rng.randint(0, 5000) for _ in counts]
    seen = torch.full((T + 2, words), 77, dtype=torch.int32, device=DEV)
    positions = torch.full((T + 2,), 77, dtype=torch.int32, device=DEV)
    ops.draft_tree(i32([p for t in trees for p in t]), i32(starts_of(counts)), i32(past), i32(counts), seen, positions, most, window)
    want, where = [], []
    for t, p in zip(trees, past):
        w, d = plain.ways(t, window)
        want.append(plain.bits(w, words))
        where += [p + x for x in d]
    assert torch.equal(seen[:T].cpu(), torch.cat(want))
    assert positions[:T].tolist() == where
    assert bool((seen[T:] == 77).all()) and bool((positions[T:] == 77).all())


def test_tree_tables_keep_to_the_rows_that_are_given():
    """Counts on the device above what the call promised, and starts outside the step, write nothing there."""
    from sleuth_b200.kernels import ops
    seen, positions = torch.full((40, 1), 77, dtype=torch.int32, device=DEV), torch.full((40,), 77, dtype=torch.int32, device=DEV)
    parents = i32([i - 1 for i in range(16)] + [0] * 4)
    ops.draft_tree(parents, i32([0, 18, -4, 20]), i32([0, 0, 0]), i32([9, 9, 3]), seen, positions, 8)
    assert seen[:8, 0].tolist() == [(1 << (i + 1)) - 1 for i in range(8)] and bool((seen[8:18] == 77).all())
    assert bool((seen[20:] == 77).all()) and bool((positions[20:] == 77).all())


# ------------------------------------------------------------------ attention ----

class Step:
    """A step with its cache: unused rows of the pools hold NaN, pages in no order, pages that no node sees taken out of the table."""

    def __init__(self, dtype, heads, kv_heads, dim, past, counts, kind="random", window=0, seed=0, sharp=1.5, bits=None):
        g = torch.Generator().manual_seed(seed)
        rng = random.Random(seed)
        self.dtype, self.heads, self.kv_heads, self.dim, self.window = dtype, heads, kv_heads, dim, window
        self.past, self.counts, self.n = list(past), list(counts), len(past)
        longest = max(p + c for p, c in zip(past, counts))
        self.stride, self.max_keys = max(1, -(-longest // 64)) + 1, max(1, longest)
        pages = self.n * self.stride + 2
        self.k = torch.full((pages, kv_heads, 64, dim), math.nan, dtype=dtype)
        self.v = torch.full((pages, kv_heads, 64, dim), math.nan, dtype=dtype)
        order = torch.randperm(pages, generator=g)
        self.table = torch.full((self.n, self.stride), -1, dtype=torch.int32)
        self.starts = starts_of(counts)
        self.T, self.words = self.starts[-1], -(-max(1, max(counts)) // 32)
        trees = [make_tree(kind, c, rng) for c in counts]
        ways = [plain.ways(t, window) for t in trees]
        self.seen = torch.cat([plain.bits(w, self.words) for w, _ in ways]) if bits is None else bits(self, g)
        self.positions = torch.tensor([p + d for p, (_, depth) in zip(past, ways) for d in depth], dtype=torch.int32)
        at = 0
        for s, (p, c) in enumerate(zip(past, counts)):
            for i in range(-(-(p + c) // 64)):
                page = int(order[at])
                at += 1
                rows = min(64, p + c - 64 * i)
                self.k[page, :, :rows] = torch.randn((kv_heads, rows, dim), generator=g).to(dtype)
                self.v[page, :, :rows] = torch.randn((kv_heads, rows, dim), generator=g).to(dtype)
                if not (window and c and 64 * i + 63 <= p - window):      # else no node sees it: a cache gives such pages back
                    self.table[s, i] = page
        self.q = (sharp * torch.randn((self.T, heads, dim), generator=g)).to(dtype)
        self.scale = dim ** -0.5

    def place(self, s, row):
        return int(self.table[s, row // 64]), row % 64

    def run(self, stream=None, promise=True, positions=True, graph=False):
        from sleuth_b200.kernels import ops
        t = [x.to(DEV) for x in (self.q, self.k, self.v)]
        tables = [i32(self.starts), i32(self.past), i32(self.counts), self.seen.to(DEV), self.positions.to(DEV), self.table.to(DEV)]
        most = max(1, max(self.counts))
        floats = ops.attention_tree_scratch_floats(self.T, self.n, most, self.heads, self.kv_heads, self.dim,
                                                   self.max_keys if promise else self.stride * 64, self.dtype)
        scratch = torch.full((max(1, floats),), math.nan, device=DEV)
        out = torch.full((self.T, self.heads * self.dim), 7.0, dtype=self.dtype, device=DEV)
        torch.cuda.synchronize()

        def call():
            ops.attention_tree(t[0], t[1], t[2], out, tables[0], tables[1], tables[2], tables[3], tables[4] if positions else None, tables[5], most, self.heads,
                               self.kv_heads, self.dim, self.window, self.scale, scratch=scratch, max_keys=self.max_keys if promise else 0, stream=stream)

        if graph:
            recorded = torch.cuda.CUDAGraph()
            with torch.cuda.graph(recorded):
                call()
            out.fill_(7.0)
            recorded.replay()
        else:
            call()
        torch.cuda.synchronize()
        assert ops.tc_status(out.device) is None or int(ops.tc_status(out.device)) == 0
        return out.cpu().view(self.T, self.heads, self.dim).double()

    def want(self):
        return plain.attention(self.q, self.k, self.v, self.starts, self.past, self.counts, self.seen, self.positions, self.table, self.heads, self.kv_heads,
                               self.window, self.scale)

    def check(self, **kw):
        out = self.run(**kw)
        want, size, slack = self.want()
        assert torch.isfinite(out).all()
        # 32-bit arithmetic as the oracle counts it; in bfloat16 also the weights' rounding and the result's, half a step (2^-8) each
        rel = slack[..., None] + ((1 + 2.0 ** -8) ** 2 - 1 if self.dtype == torch.bfloat16 else 2.0 ** -23)
        err = (out - want).abs()
        assert bool((err <= rel * size + 1e-30).all()), float((err / (rel * size + 1e-30)).max())
        return out


HEADS = [(torch.float32, 6, 3, 24), (torch.float32, 4, 4, 10), (torch.float32, 8, 2, 64), (torch.float32, 4, 2, 128), (torch.float32, 2, 1, 256),
         (torch.bfloat16, 4, 2, 64), (torch.bfloat16, 4, 1, 128), (torch.bfloat16, 6, 2, 128), (torch.bfloat16, 16, 1, 64),
         (torch.bfloat16, 3, 3, 96), (torch.bfloat16, 5, 1, 128), (torch.bfloat16, 2, 2, 128)]
IDS = [f"{str(d)[6:]}-{h}-{k}-{e}" for d, h, k, e in HEADS]


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", HEADS, ids=IDS)
@pytest.mark.parametrize("window", [0, 1, 5, 70])
@pytest.mark.parametrize("kind", ["chain", "random", "forest"])
def test_few_nodes(dtype, heads, kv_heads, dim, kind, window):
    Step(dtype, heads, kv_heads, dim, [0, 1, 59, 62, 64, 200, 130], [5, 3, 5, 7, 1, 8, 0], kind, window, seed=1).check()


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", HEADS, ids=IDS)
@pytest.mark.parametrize("window", [0, 9, 100])
def test_many_nodes(dtype, heads, kv_heads, dim, window):
    Step(dtype, heads, kv_heads, dim, [0, 70, 190, 5], [70, 33, 64, 0], "random", window, seed=2).check()


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", [HEADS[0], HEADS[5], HEADS[6], HEADS[7], HEADS[11]], ids=[IDS[i] for i in (0, 5, 6, 7, 11)])
def test_most_nodes(dtype, heads, kv_heads, dim):
    Step(dtype, heads, kv_heads, dim, [100, 3], [256, 130], "random", 0, seed=3).check()


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", [HEADS[2], HEADS[5], HEADS[6]], ids=[IDS[i] for i in (2, 5, 6)])
@pytest.mark.parametrize("past,count", [(3000, 4), (2047, 1), (1984, 64)])
def test_long_texts(dtype, heads, kv_heads, dim, past, count):
    """A few long sequences beside short ones: shares of the keys that are joined, blocks that cross sequences."""
    Step(dtype, heads, kv_heads, dim, [past, 10, past // 2 + 3], [count, count, max(1, count // 3)], "random", 0, seed=4).check()


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", [HEADS[0], HEADS[5], HEADS[6]], ids=[IDS[i] for i in (0, 5, 6)])
def test_many_sequences(dtype, heads, kv_heads, dim):
    rng = random.Random(9)
    past = [rng.choice([0, 1, 63, 64, 65, 130, rng.randint(0, 500)]) for _ in range(70)]
    Step(dtype, heads, kv_heads, dim, past, [rng.choice([0, 1, 4, 9]) for _ in past], "random", 0, seed=5).check()


def _any_bits(density):
    def make(step, g):
        b = (torch.rand((step.T, step.words * 32), generator=g) < density).long()
        words = (b.view(step.T, step.words, 32) << torch.arange(32)).sum(2)
        return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)
    return make


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", HEADS, ids=IDS)
@pytest.mark.parametrize("density", [0.0, 0.05, 1.0])
def test_any_bits(dtype, heads, kv_heads, dim, density):
    """Bits that are no tree, rows that see nothing at all (zeros), bits behind the last node."""
    step = Step(dtype, heads, kv_heads, dim, [0, 0, 60, 0], [5, 40, 9, 1], "random", 0, seed=6, bits=_any_bits(density))
    out = step.check()
    if density == 0.0:
        assert bool((out[:45] == 0).all()) and bool((out[54:] == 0).all())


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", HEADS, ids=IDS)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("window", [0, 30])
def test_what_a_node_does_not_see_never_reaches_it(dtype, heads, kv_heads, dim, bad, window):
    """Infinities and NaN in keys and values of one branch and of rows before the others' window: the other nodes' results stay the same."""
    past, counts = [61, 100, 5], [9, 40, 3]
    step = Step(dtype, heads, kv_heads, dim, past, counts, "random", window, seed=7)
    clean = step.run()
    spoilt = {}
    for s, p in enumerate(past):
        leaf = counts[s] - 1
        rows = [p + leaf] + ([max(0, p - window + 1), max(0, p - window + 2)] if window else [])
        for r in rows:
            page, at = step.place(s, r)
            for pool in (step.k, step.v):
                pool[page, :, at, ::3] = bad
        spoilt[s] = rows
    out = step.run()
    checked = 0
    for s, p in enumerate(past):
        for i in range(counts[s]):
            t = step.starts[s] + i
            lo = max(0, int(step.positions[t]) - window + 1) if window else 0
            sees = [r for r in spoilt[s] if (lo <= r < p) or (r >= p and int(step.seen[t, (r - p) // 32]) >> ((r - p) % 32) & 1)]
            if not sees:
                checked += 1
                assert torch.equal(out[t], clean[t]), (s, i)
            else:
                assert not torch.isfinite(out[t]).all()
    assert checked > 10


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", [HEADS[2], HEADS[5], HEADS[6]], ids=[IDS[i] for i in (2, 5, 6)])
def test_infinite_values_that_are_seen(dtype, heads, kv_heads, dim):
    """An infinity among the values of a branch comes out in the channels of the nodes that see it, and in no others."""
    step = Step(dtype, heads, kv_heads, dim, [20], [12], "random", 0, seed=8)
    page, at = step.place(0, 20 + 3)
    step.v[page, :, at, 1] = math.inf
    out = step.run()
    for t in range(12):
        hit = bool(int(step.seen[t, 0]) >> 3 & 1)
        assert bool((out[t, :, 1] == math.inf).all()) == hit
        assert torch.isfinite(out[t][:, [0] + list(range(2, dim))]).all()


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", [HEADS[2], HEADS[5], HEADS[6]], ids=[IDS[i] for i in (2, 5, 6)])
def test_queries_that_are_no_numbers_spoil_their_own_rows(dtype, heads, kv_heads, dim):
    step = Step(dtype, heads, kv_heads, dim, [150, 20], [12, 30], "random", 0, seed=8)
    clean = step.run()
    step.q[5] = math.nan
    step.q[20, 0] = math.inf
    out = step.run()
    for t in range(42):
        for h in range(heads):
            if t == 5 or (t == 20 and h == 0):
                assert not torch.isfinite(out[t, h]).any()
            else:
                assert torch.equal(out[t, h], clean[t, h])


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", [HEADS[0], HEADS[5], HEADS[6], HEADS[7]], ids=[IDS[i] for i in (0, 5, 6, 7)])
def test_streams_graphs_promises(dtype, heads, kv_heads, dim):
    step = Step(dtype, heads, kv_heads, dim, [300, 64, 0], [6, 20, 2], "random", 0, seed=10)
    out = step.check()
    side = torch.cuda.Stream()
    assert torch.equal(step.run(stream=side.cuda_stream), out)
    assert torch.equal(step.run(graph=True), out)
    assert torch.equal(step.run(positions=False), out)
    step.check(promise=False)


def test_long_window_and_large_positions():
    step = Step(torch.bfloat16, 4, 2, 128, [200, 3], [6, 20], "random", 2 ** 31 - 1, seed=11)
    whole = Step(torch.bfloat16, 4, 2, 128, [200, 3], [6, 20], "random", 0, seed=11)
    assert torch.equal(step.run(), whole.run())
    step.positions += 2 ** 31 - 1 - int(step.positions.max())      # far positions under a short window: nothing from before the step is left
    step.window = 5
    out = step.run()
    none = Step(torch.bfloat16, 4, 2, 128, [0, 0], [6, 20], "random", 0, seed=11)
    assert torch.isfinite(out).all() and none.T == step.T


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", [HEADS[0], HEADS[5], HEADS[6]], ids=[IDS[i] for i in (0, 5, 6)])
def test_pages_that_the_pool_has_not_read_as_zeros(dtype, heads, kv_heads, dim):
    step = Step(dtype, heads, kv_heads, dim, [200, 70], [5, 9], "random", 0, seed=12)
    for s, i, bad in ((0, 1, -1), (0, 2, 10 ** 6), (1, 0, step.k.shape[0])):
        page = int(step.table[s, i])
        step.k[page], step.v[page] = 0, 0
        step.table[s, i] = bad
    out = step.run()
    for s, i in ((0, 1), (0, 2), (1, 0)):      # what the oracle reads there: pages of zeros
        step.table[s, i] = step.k.shape[0]
    step.k, step.v = (torch.cat([t, torch.zeros_like(t[:1])]) for t in (step.k, step.v))
    want, size, slack = step.want()
    rel = slack[..., None] + ((1 + 2.0 ** -8) ** 2 - 1 if dtype == torch.bfloat16 else 2.0 ** -23)
    assert bool(((out - want).abs() <= rel * size + 1e-30).all())


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", [HEADS[0], HEADS[5], HEADS[6]], ids=[IDS[i] for i in (0, 5, 6)])
def test_page_numbers_whose_rows_pass_32_bits_read_as_zeros(dtype, heads, kv_heads, dim):
    """A number of pages that, times the rows of a page, comes round to the pool's own ones in 32 bits."""
    step = Step(dtype, heads, kv_heads, dim, [200, 70], [5, 9], "random", 0, seed=12)
    around = 2 ** 26 // (kv_heads & -kv_heads)
    for s, i in ((0, 1), (1, 0)):
        page = int(step.table[s, i])
        step.table[s, i] = page + around
    out = step.run()
    for s, i in ((0, 1), (1, 0)):
        step.table[s, i] = step.k.shape[0]
    step.k, step.v = (torch.cat([t, torch.zeros_like(t[:1])]) for t in (step.k, step.v))
    want, size, slack = step.want()
    rel = slack[..., None] + ((1 + 2.0 ** -8) ** 2 - 1 if dtype == torch.bfloat16 else 2.0 ** -23)
    assert bool(((out - want).abs() <= rel * size + 1e-30).all())


def test_counts_beyond_the_given_tokens_write_nothing_there():
    from sleuth_b200.kernels import ops
    for dtype in (torch.float32, torch.bfloat16):
        q, pool = torch.randn((6, 2, 64), device=DEV).to(dtype), torch.randn((3, 1, 64, 64), device=DEV).to(dtype)
        memory = torch.full((9, 128), 7.0, dtype=dtype, device=DEV)
        seen = torch.full((6, 1), -1, dtype=torch.int32, device=DEV)
        floats = ops.attention_tree_scratch_floats(6, 3, 8, 2, 1, 64, 64, dtype)
        scratch = torch.zeros(max(1, floats), device=DEV)
        ops.attention_tree(q, pool, pool, memory[:6], i32([0, 4, 30]), i32([3, 3, 3]), i32([4, 8, 8]), seen, None, i32([[0], [1], [2]]), 8, 2, 1, 64, 0, 0.1, scratch=scratch)
        assert bool((memory[6:] == 7.0).all()) and torch.isfinite(memory).all() and not bool((memory[:6] == 7.0).all(1).any())


class Elsewhere(torch.Tensor):
    def get_device(self):
        return 5


def moved(a, moved=None, **kw):
    a = {**a, **kw}
    return a if moved is None else {**a, moved: a[moved].as_subclass(Elsewhere)}


def test_refused_calls():
    from sleuth_b200.kernels import ops
    z = lambda *shape, t=torch.int32: torch.zeros(shape, dtype=t, device=DEV)  # noqa: E731
    bf, f32 = torch.bfloat16, torch.float32

    def attention(error, match, **kw):
        a = dict(q=z(4, 4, 64, t=bf), k_pool=z(2, 2, 64, 64, t=bf), v_pool=z(2, 2, 64, 64, t=bf), out=z(4, 256, t=bf), seq_start=z(1), past=z(1), counts=z(1), seen=z(4, 1),
                 positions=z(4), block_table=z(1, 2), max_count=4, heads=4, kv_heads=2, head_dim=64, window=0, scale=0.1, scratch=z(1 << 20, t=f32))
        with pytest.raises(error, match=match):
            ops.attention_tree(**moved(a, **kw))

    attention(ValueError, "contiguous", q=z(4, 4, 128, t=bf)[..., ::2])
    attention(ValueError, "alike", out=z(4, 256, t=f32))
    attention(ValueError, "pools", v_pool=z(2, 2, 64, 32, t=bf))
    attention(ValueError, "heads", heads=8)
    attention(ValueError, "nodes", max_count=257, seen=z(4, 9))
    attention(ValueError, "bit", max_count=33)
    attention(ValueError, "int32", counts=z(1, t=torch.int64))
    attention(ValueError, "positions", window=5, positions=None)
    attention(ValueError, "window", window=-1)
    attention(ValueError, "scale", scale=0.0)
    attention(ValueError, "range", window=2 ** 31)
    attention(ValueError, "range", max_keys=2 ** 40)
    attention(RuntimeError, "scratch", scratch=None, max_keys=0, block_table=z(1, 4000))
    attention(RuntimeError, "heads", q=z(4, 3, 64, t=bf), heads=3, out=z(4, 192, t=bf))
    attention(RuntimeError, "head_dim", q=z(4, 4, 65, t=f32), k_pool=z(2, 2, 64, 65, t=f32), v_pool=z(2, 2, 64, 65, t=f32), out=z(4, 260, t=f32), head_dim=65)
    attention(RuntimeError, "aligned", q=z(4 * 4 * 64 + 1, t=bf)[1:].view(4, 4, 64))

    def tree(match, **kw):
        a = dict(parents=z(4), seq_start=z(2), past=z(1), counts=z(1), seen=z(4, 1), positions=z(4), max_count=4)
        with pytest.raises(ValueError, match=match):
            ops.draft_tree(**moved(a, **kw))

    tree("int32", parents=z(4, t=torch.int64))
    tree("row a sequence", counts=z(2))
    tree("bit", seen=z(3, 1))
    tree("bit", max_count=40)
    tree("nodes", max_count=0)
    tree("window", window=-3)
    tree("range", window=2 ** 31)
    tree("contiguous", seen=z(4, 2)[:, :1])

    def verify(match, error=ValueError, **kw):
        a = dict(logits=z(4, 50, t=f32), limit=50, tokens=z(4), parents=z(4), seq_start=z(1), counts=z(1), uniforms=z(4, t=f32), temperature=1.0, path=z(1, 4), lengths=z(1), chosen=z(1),
                 max_count=4, scratch=z(100))
        with pytest.raises(error, match=match):
            ops.verify_drafts(**moved(a, **kw))

    verify("limit", limit=51)
    verify("limit", probs=z(3, 50, t=f32))
    verify("float32", logits=z(4, 50, t=bf))
    verify("stride", logits=z(4, 100, t=f32)[:, ::2])
    verify("temperature", temperature=math.inf)
    verify("temperature", temperature=math.nan)
    verify("uniforms", uniforms=None)
    verify("floors", floors=z(3, t=f32))
    verify("path", path=z(1, 3))
    verify("nodes", max_count=300, path=z(1, 300))
    verify("int32", tokens=z(4, t=torch.int64))
    verify("value for each", tokens=z(3))
    verify("scratch", error=RuntimeError, scratch=None)

    def compact(match, **kw):
        a = dict(k_pool=z(2, 2, 1, 64, 8, t=bf), block_table=z(1, 2), past=z(1), path=z(1, 4), lengths=z(1))
        with pytest.raises(ValueError, match=match):
            ops.cache_compact(**moved(a, **kw))

    compact("pools", k_pool=z(2, 1, 32, 8, t=bf))
    compact("four", k_pool=z(2, 1, 64, 7, t=bf))
    compact("v_pool", v_pool=z(3, 1, 64, 8, t=bf))
    compact("at most", path=z(1, 257))
    compact("int32", past=z(1, t=torch.int64))
    compact("contiguous", k_pool=z(2, 1, 64, 16, t=bf)[..., :8])
    # one tensor after the other on another device (these say so alone)
    for name in ("k_pool", "v_pool", "out", "seq_start", "past", "counts", "seen", "positions", "block_table", "scratch"):
        attention(ValueError, "device", moved=name)
    for name in ("seq_start", "past", "counts", "seen", "positions"):
        tree("device", moved=name)
    for name in ("probs", "tokens", "parents", "seq_start", "counts", "uniforms", "floors", "path", "lengths", "chosen", "scratch"):
        verify("device", moved=name, probs=z(4, 50, t=f32), floors=z(4, t=f32))
    for name in ("v_pool", "block_table", "past", "path", "lengths"):
        compact("device", moved=name, v_pool=z(2, 2, 1, 64, 8, t=bf))
    # nothing to do is no mistake
    ops.draft_tree(z(0), z(1), z(0), z(0), z(0, 1), z(0), 1)
    ops.cache_compact(z(2, 1, 64, 8, t=bf), z(0, 2), z(0), z(0, 4), z(0))
    ops.verify_drafts(z(0, 50, t=f32), 50, z(0), z(0), z(0), z(0), z(0, t=f32), 1.0, z(0, 4), z(0), z(0), 4)
    lengths, chosen, path = z(2) + 9, z(2) + 9, z(2, 4) + 9
    ops.verify_drafts(z(0, 50, t=f32), 50, z(0), z(0), z(3), z(2), z(0, t=f32), 1.0, path, lengths, chosen, 4)
    assert lengths.tolist() == [0, 0] and chosen.tolist() == [-1, -1] and bool((path == -1).all())
    ops.attention_tree(z(0, 4, 64, t=bf), z(2, 2, 64, 64, t=bf), z(2, 2, 64, 64, t=bf), z(0, 256, t=bf), z(1), z(0), z(0), z(0, 1), None, z(0, 2), 4, 4, 2, 64, 0, 0.1)


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", HEADS, ids=IDS)
@pytest.mark.parametrize("past,counts", [([0, 10, 60], [3, 6, 5]), ([700, 70], [4, 9]), ([0, 40] * 40, [2, 5] * 40), ([90, 5], [130, 140])], ids=["few", "long", "many", "broad"])
def test_results_are_off_by_their_own_rounding(dtype, heads, kv_heads, dim, past, counts):
    """In bfloat16 a result is rounded once, by half a step (2^-8 of it); weights are off by 2^-14 at most (two parts of 16 bits, the first up to two steps of 2^-7
    below the weight, the second cut to eight digits: 2^-6 2^-8), beside what 32-bit sums leave (the oracle's slack)."""
    step = Step(dtype, heads, kv_heads, dim, past, counts, "random", 0, seed=30)
    out = step.run()
    want, size, slack = step.want()
    own, weights = (2.0 ** -8, 2.0 ** -14) if dtype == torch.bfloat16 else (2.0 ** -24, 2.0 ** -23)
    err, allowed = (out - want).abs(), (slack[..., None] + weights) * size
    assert bool((err <= allowed * (1 + own) + own * want.abs() + 1e-30).all()), float((err / (allowed + own * want.abs() + 1e-30)).max())


def _scores(step, q0, k0, k1, twins):
    """Every node sees the rows before the step, whose scores lie far below, and of the step's own rows itself (with ``twins`` the node beside it too); its score
    there is q0 k0 + k1."""
    step.q.zero_()
    step.q[..., 0], step.q[..., 1] = q0, 1.0
    rows = torch.isfinite(step.k)
    step.k[rows] = 0.0
    for s, (p, c) in enumerate(zip(step.past, step.counts)):
        for r in range(p + c):
            page, at = step.place(s, r)
            step.k[page, :, at, 0] = k0 if r >= p else 2 * k0 if k0 < 0 else k0 / 2
            step.k[page, :, at, 1] = k1 if r >= p else 0.0
    want = torch.zeros((step.T, step.heads, step.dim), dtype=torch.float64)
    for s, (p, c) in enumerate(zip(step.past, step.counts)):
        for i in range(c):
            seen = [i, i ^ 1] if twins and i ^ 1 < c else [i]
            word = torch.zeros(step.words * 32, dtype=torch.int64)
            word[seen] = 1
            word = (word.view(-1, 32) << torch.arange(32)).sum(1)
            step.seen[step.starts[s] + i] = torch.where(word >= 1 << 31, word - (1 << 32), word).to(torch.int32)
            values = [step.v[step.place(s, p + b)[0], :, step.place(s, p + b)[1]].double() for b in seen]
            want[step.starts[s] + i] = (sum(values) / len(values)).repeat_interleave(step.heads // step.kv_heads, 0)
    return want


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", [HEADS[2], HEADS[5], HEADS[6], HEADS[9]], ids=[IDS[i] for i in (2, 5, 6, 9)])
@pytest.mark.parametrize("past,counts", [([0, 30, 200], [3, 6, 5]), ([3000, 70], [4, 9]), ([0, 100] * 40, [2, 5] * 40), ([90, 5], [130, 140])],
                         ids=["few", "long", "many", "broad"])
@pytest.mark.parametrize("q0,k0,k1", [(512.0, 256.0, 1.0), (512.0, -256.0, -1020.0), (2048.0, 128.0, 56.0), (2.0 ** 20, 2.0 ** 12, 255 * 2.0 ** 17), (2.0 ** 20, -2.0 ** 12, -255 * 2.0 ** 17),
                                      (2.0 ** 30, 2.0 ** 30, 255 * 2.0 ** 45), (2.0 ** 30, -2.0 ** 30, -255 * 2.0 ** 45)])
def test_large_scores(dtype, heads, kv_heads, dim, past, counts, q0, k0, k1):
    """Scores of 10^4 to 10^17, of both signs, just above and just below what 16 bits hold: a node that sees one key of such a score gives that key's value as it
    is; two of the same score, their mean."""
    step = Step(dtype, heads, kv_heads, dim, past, counts, "star", 0, seed=31)
    want = _scores(step, q0, k0, k1, False)
    assert torch.equal(step.run(), want)
    want = _scores(step, q0, k0, k1, True)
    # half a step of the result; a float32 sum's and quotient's, weights' parts (2^-14 of a weight, the same for both)
    rounding = 2.0 ** -8 + 2.0 ** -13 if dtype == torch.bfloat16 else 2.0 ** -23
    assert bool(((step.run() - want).abs() <= rounding * want.abs() + 1e-30).all())


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", [HEADS[0], HEADS[2], HEADS[5], HEADS[6], HEADS[9]], ids=[IDS[i] for i in (0, 2, 5, 6, 9)])
def test_tables_that_the_kernel_in_front_writes(dtype, heads, kv_heads, dim):
    """The numbers of rows and nodes come from a judgement right in front of the attention, which lets it begin early: always the new ones count."""
    from sleuth_b200.kernels import ops
    vocab, n, most = 4000, 6, 6
    past, counts = [700, 300, 5, 0, 64, 1000], [6, 5, 4, 3, 2, 1]
    step = Step(dtype, heads, kv_heads, dim, past, counts, "chain", 0, seed=32)
    t = [x.to(DEV) for x in (step.q, step.k, step.v)]
    starts, seen, table = i32(step.starts), step.seen.to(DEV), step.table.to(DEV)
    floats = ops.attention_tree_scratch_floats(step.T, n, most, heads, kv_heads, dim, step.stride * 64, dtype)
    assert floats > 0 or dtype == torch.bfloat16 and dim in (64, 128)
    scratch = torch.zeros(max(1, floats), device=DEV)
    # a judgement whose lengths are the counts: greedy chains of which the first counts[s] nodes are right
    logits = torch.zeros((n * most, vocab), device=DEV)
    logits[:, 7] = 1.0
    tokens = torch.full((n, most), 7, dtype=torch.int32)
    for s, c in enumerate(counts):
        tokens[s, c:] = 8
    tokens = tokens.view(-1).to(DEV)
    parents, verify_starts, sixes = i32([i - 1 for i in range(most)] * n), i32([most * s for s in range(n)]), i32([most] * n)
    path, lengths, chosen = (torch.zeros(s, dtype=torch.int32, device=DEV) for s in ((n, most), (n,), (n,)))
    words = torch.zeros(max(1, ops.verify_drafts_scratch_words(n, n * most, vocab, False)), dtype=torch.int32, device=DEV)
    # and a tree table whose positions are the numbers of rows before the step: trees of single nodes
    pasts, single, ones = i32([0] * n), i32([-1] * n), i32([1] * n)
    bits, before = torch.zeros((n, 1), dtype=torch.int32, device=DEV), i32(past)
    out = torch.empty((step.T, heads * dim), dtype=dtype, device=DEV)
    wanted = step.run(promise=False).view(step.T, -1)

    def call():
        ops.verify_drafts(logits, vocab, tokens, parents, verify_starts, sixes, None, 0.0, path, lengths, chosen, most, scratch=words)
        ops.draft_tree(single, i32_range, before, ones, bits, pasts, 1)
        ops.attention_tree(t[0], t[1], t[2], out, starts, pasts, lengths, seen, None, table, most, heads, kv_heads, dim, 0, step.scale, scratch=scratch)

    i32_range = i32(list(range(n)))
    graph = torch.cuda.CUDAGraph()
    call()
    torch.cuda.synchronize()
    assert lengths.tolist() == counts and pasts.tolist() == past
    with torch.cuda.graph(graph):
        for _ in range(4):
            call()
    for again in range(20):
        lengths.fill_(again % 3)
        pasts.fill_(again)
        out.fill_(7.0)
        graph.replay() if again % 2 else call()
        assert torch.equal(out.cpu().double(), wanted), again


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", [HEADS[0], HEADS[2], HEADS[5], HEADS[6], HEADS[9]], ids=[IDS[i] for i in (0, 2, 5, 6, 9)])
@pytest.mark.parametrize("window", [1, 5, 150, 2 ** 31 - 1])
@pytest.mark.parametrize("far", [0, 3, 140, 2 ** 31])
def test_positions_far_from_their_rows(dtype, heads, kv_heads, dim, window, far):
    """Positions up to the last of 32 bits, far beyond the rows: what lies before the step and in the window is what counts, nothing where the window is short."""
    step = Step(dtype, heads, kv_heads, dim, [200, 3], [6, 20], "random", 0, seed=11)
    step.window = window
    step.positions += min(far, 2 ** 31 - 1 - int(step.positions.max()))
    step.check()


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", [HEADS[2], HEADS[5], HEADS[6], HEADS[8], HEADS[9]], ids=[IDS[i] for i in (2, 5, 6, 8, 9)])
@pytest.mark.parametrize("past,counts", [([200], [12]), ([400, 70] * 40, [3, 5] * 40), ([130, 64], [40, 256])], ids=["few", "many", "broad"])
@pytest.mark.parametrize("sharp", [0.0, 1.5])
def test_infinite_values_before_the_step(dtype, heads, kv_heads, dim, past, counts, sharp):
    """An infinity among the values of a row that every node sees comes out in its channel, whatever its weight (where all scores are equal every weight is 1 and has
    no second part), and leaves the other channels alone."""
    step = Step(dtype, heads, kv_heads, dim, past, counts, "random", 0, seed=33, sharp=sharp)
    clean = step.run()
    for s, p in enumerate(past):
        for row, channel, value in ((10, 1, math.inf), (p - 1, dim - 1, -math.inf)):
            page, at = step.place(s, row)
            step.v[page, :, at, channel] = value
    out = step.run()
    assert bool((out[..., 1] == math.inf).all()) and bool((out[..., dim - 1] == -math.inf).all())
    assert torch.equal(out[..., 2:dim - 1], clean[..., 2:dim - 1]) and torch.equal(out[..., 0], clean[..., 0])


# ------------------------------------------------------------------ verification ----

class Judged:
    def __init__(self, counts, kind, vocab, limit, temperature, drawn, floors=False, seed=0, pad=0, sharp=2.0):
        g = torch.Generator().manual_seed(seed)
        rng = random.Random(seed)
        self.counts, self.vocab, self.limit, self.temperature = counts, vocab, limit, temperature
        self.starts, self.trees = starts_of(counts), [make_tree(kind, c, rng) for c in counts]
        T = self.starts[-1]
        self.pad = pad
        common = sharp * torch.randn((T, vocab + pad), generator=g)
        self.logits = common + 0.8 * torch.randn((T, vocab + pad), generator=g)
        draft = torch.softmax((common + 0.8 * torch.randn((T, vocab + pad), generator=g))[:, :limit] / (temperature or 1.0), 1)
        self.probs = torch.zeros((T, vocab + pad))
        self.probs[:, :limit] = draft
        self.tokens = torch.zeros(T, dtype=torch.int32)
        for s, tree in enumerate(self.trees):
            for j, p in enumerate(tree):
                if 0 <= p < j:
                    at = self.starts[s] + p
                    pick = torch.multinomial(draft[at], 1, generator=g) if drawn else torch.topk(self.logits[at, :limit], min(3, limit)).indices[rng.randrange(min(3, limit))]
                    self.tokens[self.starts[s] + j] = int(pick)
        self.uniforms = torch.rand(T, generator=g)
        self.floors = torch.topk(self.logits[:, :limit], min(limit, 20), dim=1).values[:, -1].contiguous() if floors else None
        if not drawn:
            self.probs = None

    def run(self, stream=None, width=0, graph=False):
        from sleuth_b200.kernels import ops
        n, T, most = len(self.counts), self.starts[-1], max(1, max(self.counts))
        width = width or most
        dev = lambda t: None if t is None else t.to(DEV)  # noqa: E731
        logits, probs = dev(self.logits)[:, :self.vocab], dev(self.probs)
        probs = None if probs is None else probs[:, :self.vocab]
        parents = i32([p for t in self.trees for p in t])
        path, lengths, chosen = (torch.full(s, 99, dtype=torch.int32, device=DEV) for s in ((n, width), (n,), (n,)))
        args = (logits, self.limit, dev(self.tokens), parents, i32(self.starts), i32(self.counts), dev(self.uniforms), self.temperature, path, lengths, chosen, most)
        words = ops.verify_drafts_scratch_words(n, T, self.limit, probs is not None)
        kw = dict(probs=probs, floors=dev(self.floors), scratch=torch.full((max(1, words),), -1, dtype=torch.int32, device=DEV), stream=stream)
        torch.cuda.synchronize()
        if graph:
            recorded = torch.cuda.CUDAGraph()
            with torch.cuda.graph(recorded):
                ops.verify_drafts(*args, **{**kw, "stream": None})
            for t in (path, lengths, chosen):
                t.fill_(99)
            recorded.replay()
        else:
            ops.verify_drafts(*args, **kw)
        torch.cuda.synchronize()
        return path.cpu(), lengths.cpu(), chosen.cpu()

    def check(self, **kw):
        path, lengths, chosen = self.run(**kw)
        for s, c in enumerate(self.counts):
            at = slice(self.starts[s], self.starts[s + 1])
            want, token = plain.verify(self.logits[at], self.tokens[at], self.trees[s], self.uniforms[at], self.temperature, self.limit,
                                       None if self.probs is None else self.probs[at], None if self.floors is None else self.floors[at])
            assert path[s].tolist() == want + [-1] * (path.shape[1] - len(want)), (s, path[s].tolist(), want)
            assert int(lengths[s]) == len(want) and int(chosen[s]) == token, (s, int(chosen[s]), token)
        return path, lengths, chosen


@pytest.mark.parametrize("vocab,limit,pad", [(5, 5, 0), (300, 257, 3), (1000, 1000, 0), (4096, 4095, 8), (33000, 32999, 1)])
@pytest.mark.parametrize("temperature", [0.0, 0.4, 1.0, 3.0])
@pytest.mark.parametrize("kind,drawn,floors", [("chain", True, False), ("random", True, False), ("random", False, False), ("star", True, True), ("random", False, True),
                                               ("forest", False, False), ("star", False, False)])
def test_verification(vocab, limit, pad, temperature, kind, drawn, floors):
    Judged([5, 1, 0, 9, 17, 2, 8], kind, vocab, limit, temperature, drawn, floors, seed=vocab + int(10 * temperature), pad=pad).check()


def _beside(border):
    """The nearest float32 numbers below and above, further away than what the sums leave open (1e-11)."""
    down = torch.tensor(border, dtype=torch.float32)
    while float(down) > border * (1 - 1e-10):
        down = torch.nextafter(down, torch.tensor(0.0))
    up = torch.nextafter(down, torch.tensor(2.0))
    while float(up) < border * (1 + 1e-10):
        up = torch.nextafter(up, torch.tensor(2.0))
    return down, up


@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("temperature", [0.01, 0.02, 0.3, 1.0, 30.0])
@pytest.mark.parametrize("vocab,wanted", [(40, 0.9), (4100, 0.6), (30000, 0.02)])
def test_numbers_next_to_a_probability(vocab, wanted, temperature, drawn):
    """Random numbers that are the nearest float32 below and above a draft's probability (over that of its draw): accepted and refused, as in 64 bits. Where a second
    child follows, the refused one's probability counts as exactly."""
    n = 120
    counts = [3] * n
    j = Judged(counts, "star", vocab, vocab, temperature, drawn, seed=41)
    g = torch.Generator().manual_seed(41)
    T = 3 * n
    j.logits = 20.0 + 3.0 * temperature * torch.randn((T, vocab), generator=g)
    if drawn:
        j.probs = torch.softmax(torch.randn((T, vocab), generator=g), 1)
    for s in range(n):
        row = j.logits[3 * s]
        x, y = s % vocab, (s + 7) % vocab
        # token x gets about the wanted share of the row, y half of what is left where it is the second child's turn
        for token, share in ((x, wanted), (y, 0.5 * (1 - wanted) if s % 4 > 1 else 0.1 * wanted)):
            rest = torch.logsumexp(torch.cat([row[:token], row[token + 1:]]).double() / temperature, 0)
            row[token] = float((rest + math.log(share / (1 - share))) * temperature)
        p = torch.softmax(row.double() / temperature, 0)
        j.tokens[3 * s + 1], j.tokens[3 * s + 2] = x, y
        if drawn:
            q = j.probs[3 * s].double()
            q[x] = min(1.0, float(p[x]) * 1.3)
            j.probs[3 * s] = q.float()
        border = float(p[x]) / (float(j.probs[3 * s, x]) if drawn else 1.0)
        down, up = _beside(border)
        if s % 4 > 1 and not drawn:      # the first is refused, the second lies at its border
            j.uniforms[3 * s + 1] = 1.0 - 2.0 ** -24
            down, up = _beside(float(p[y]) / (1.0 - float(p[x])))
            j.uniforms[3 * s + 2] = down if s % 2 else up
        else:
            j.uniforms[3 * s + 1] = down if s % 2 else up
            j.uniforms[3 * s + 2] = 0.9
    j.check()


@pytest.mark.parametrize("drawn", [True, False])
def test_verification_of_a_large_vocabulary(drawn):
    Judged([6, 6, 4, 1], "chain", 151936, 151936, 0.8, drawn, seed=3, sharp=2.5).check()


def test_verification_of_many_sequences_and_nodes():
    rng = random.Random(4)
    Judged([rng.choice([1, 2, 5, 6]) for _ in range(200)], "random", 500, 500, 1.0, True, seed=5).check()
    Judged([256, 255, 100], "random", 64, 64, 1.0, False, seed=6).check()
    Judged([256, 33], "star", 400, 400, 1.5, True, seed=7).check()
    Judged([256], "chain", 8, 8, 0.0, False, seed=8).check()


@pytest.mark.parametrize("temperature", [0.0, 1.0, 1e-40, 1e300])
def test_verification_of_odd_logits(temperature):
    """NaN and -inf have no probability, an infinite logit all of it, a row of nothing picks token 0."""
    j = Judged([4, 4, 4, 4, 4], "chain", 400, 400, temperature, False, seed=9)
    j.logits[:, 5::7] = math.nan
    j.logits[:, 6::7] = -math.inf
    j.logits[0, 100] = math.inf
    j.tokens[1] = 100
    j.logits[4:8] = -math.inf
    j.logits[8:12, 1:] = math.nan
    j.tokens[9:12] = 0
    j.tokens[13:15] = torch.tensor([400, -1], dtype=torch.int32)
    path, lengths, chosen = j.check()
    assert int(lengths[0]) >= 2 and int(chosen[1]) == 0 and int(lengths[2]) == 4 and int(lengths[3]) == 1


def test_rows_without_a_number_above_minus_infinity_pick_token_0():
    """Whether the row has children or not, and whatever stands in front of the first -inf."""
    j = Judged([3, 1, 2], "chain", 300, 300, 0.0, False, seed=9)
    j.logits[:] = -math.inf
    j.logits[:, :3] = math.nan
    j.tokens[:] = 3
    path, lengths, chosen = j.run()
    assert chosen.tolist() == [0, 0, 0] and lengths.tolist() == [1, 1, 1]


@pytest.mark.parametrize("temperature", [0.0, 0.7])
@pytest.mark.parametrize("drawn", [True, False])
def test_verification_of_masked_rows(temperature, drawn):
    """Rows most of whose tokens carry the type's lowest value, one of them all; a floor above every logit leaves nothing."""
    j = Judged([5, 5, 3, 4], "random", 20000, 20000, temperature, drawn, seed=11)
    lowest = torch.finfo(torch.float32).min
    allowed = torch.zeros(20000, dtype=torch.bool)
    allowed[torch.randperm(20000, generator=torch.Generator().manual_seed(3))[:40]] = True
    allowed[j.tokens[1:3].long()] = True
    j.logits[:5, ~allowed] = lowest
    j.logits[5:10, 12000:] = lowest
    j.logits[10:13] = lowest
    if temperature:
        j.floors = torch.full((17,), -50.0)
        j.floors[10:13] = -math.inf
        j.floors[13:] = 1e9
    path, lengths, chosen = j.check()
    assert bool(allowed[int(chosen[0])]) and (not temperature or (int(lengths[3]) == 1 and int(chosen[3]) == 0))


def test_verification_streams_graphs_widths():
    j = Judged([6, 3, 9], "random", 2000, 2000, 0.9, True, seed=10)
    first = j.check()
    for again in (j.run(stream=torch.cuda.Stream().cuda_stream), j.run(graph=True)):
        assert all(torch.equal(a, b) for a, b in zip(first, again))
    j.check(width=12)


@pytest.mark.parametrize("drawn", [True, False])
def test_verified_tokens_follow_the_target(drawn):
    """Whatever the drafts are, the first token behind node 0 is distributed as the target says: 20,000 trees of one row of logits each,
    counts within five standard deviations."""
    n, vocab, width = 20000, 7, 3
    g = torch.Generator().manual_seed(12)
    target, draft = torch.tensor([2.0, 1.0, 0.0, 1.5, -1.0, 0.3, -3.0]), torch.softmax(torch.tensor([0.0, 2.0, 0.5, 1.0, 1.0, -1.0, -8.0]), 0)
    j = Judged([1 + width] * n, "star", vocab, vocab, 1.0, True, seed=13)
    j.logits = target.repeat(n * (1 + width), 1).contiguous()
    j.probs = draft.repeat(n * (1 + width), 1).contiguous() if drawn else None
    j.tokens = torch.multinomial(draft, n * (1 + width), replacement=True, generator=g).to(torch.int32) if drawn else \
        torch.tensor([0, 1, 4, 1], dtype=torch.int32).repeat(n)
    path, lengths, chosen = j.run()
    first = torch.where(lengths > 1, j.tokens.view(n, 1 + width).gather(1, path[:, 1:2].clamp(min=0).long())[:, 0], chosen)
    counts, p = torch.bincount(first.long(), minlength=vocab).double(), torch.softmax(target.double(), 0)
    assert bool(((counts - n * p).abs() <= 5 * (n * p * (1 - p)).sqrt() + 1).all()), (counts / n, p)


# ------------------------------------------------------------------ compaction ----

@pytest.mark.parametrize("dtype,layers,kv_heads,dim,vdim", [(torch.bfloat16, (3, 2), 2, 128, 0), (torch.bfloat16, (), 3, 10, 0), (torch.float32, (2,), 3, 24, 0),
                                                            (torch.bfloat16, (2,), 1, 64, 128), (torch.float32, (), 2, 7, 9), (torch.bfloat16, (1,), 2, 6, 64)])
def test_compaction(dtype, layers, kv_heads, dim, vdim):
    from sleuth_b200.kernels import ops
    rng = random.Random(dim)
    past, counts = [0, 60, 64, 127, 3, 10, 5], [6, 40, 64, 9, 1, 0, 256]
    paths = [sorted(rng.sample(range(c), rng.randint(1, c))) if c else [] for c in counts]
    paths[0], paths[1] = [0, 2, 3, 4, 5], list(range(1, 40))        # sources that are targets of the row after
    stride = 6
    pages = len(past) * stride + 1
    table = torch.randperm(pages)[:len(past) * stride].to(torch.int32).view(len(past), stride)
    k = torch.randn((*layers, pages, kv_heads, 64, dim)).to(dtype)
    v = torch.randn((*layers, pages, kv_heads, 64, vdim)).to(dtype) if vdim else None
    path = torch.full((len(past), 256), -1, dtype=torch.int32)
    for s, p in enumerate(paths):
        path[s, :len(p)] = torch.tensor(p, dtype=torch.int32)
    kd, vd = k.to(DEV), None if v is None else v.to(DEV)
    ops.cache_compact(kd, table.to(DEV), i32(past), path.to(DEV), i32([len(p) for p in paths]), v_pool=vd)
    for pool, got in ((k, kd), (v, vd)):
        if pool is not None:
            plain.compact(pool.view(-1, *pool.shape[-4:]), table, past, paths)
            assert torch.equal(got.cpu(), pool)


def test_compaction_ends_where_a_path_does_not_rise():
    from sleuth_b200.kernels import ops
    pool = torch.randn((2, 3, 1, 64, 8))
    table = torch.tensor([[0], [1], [2]], dtype=torch.int32)
    path = torch.tensor([[0, 2, 2, 5], [1, 3, -1, 9], [0, 4, 70, 71]], dtype=torch.int32)
    got = pool.to(DEV)
    ops.cache_compact(got, table.to(DEV), i32([10, 0, 5]), path.to(DEV), i32([4, 9, 4]))
    plain.compact(pool, table, [10, 0, 5], [[0, 2], [1, 3], [0, 4]])
    assert torch.equal(got.cpu(), pool)
    # nor where a row lies on a page that the pool has not
    pool = torch.randn((2, 3, 1, 64, 8))
    table = torch.tensor([[0, -1], [1, 3], [2, 0]], dtype=torch.int32)
    path = torch.tensor([[0, 2, 3, 20], [1, 9, 10, 11], [0, 3, 9, 10]], dtype=torch.int32)
    got = pool.to(DEV)
    ops.cache_compact(got, table.to(DEV), i32([60, 57, 60]), path.to(DEV), i32([4, 4, 4]))
    plain.compact(pool, table, [60, 57, 60], [[0, 2, 3], [1], [0, 3, 9, 10]])
    assert torch.equal(got.cpu(), pool)


# ------------------------------------------------------------------ together ----

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_step_of_drafted_tokens_and_the_step_after_it(dtype):
    """Tree tables, attention, verification and compaction one after the other, recorded as one graph; then a single-token step over what is left of the
    cache: its attention is that of the accepted tokens alone."""
    from sleuth_b200.kernels import ops
    heads, kv_heads, dim, vocab = 8, 4, 64, 700
    past, counts = [70, 5, 128], [9, 4, 12]
    step = Step(dtype, heads, kv_heads, dim, past, counts, "random", 0, seed=21)
    rng = random.Random(21)
    j = Judged(counts, "random", vocab, vocab, 1.0, True, seed=21)
    trees = [make_tree("random", c, rng) for c in counts]
    j.trees = trees
    T, n, most, stride = step.T, 3, max(counts), step.stride
    dev = lambda t: t.to(DEV)  # noqa: E731
    q, k, v, table = map(dev, (step.q, step.k, step.v, step.table))
    parents, starts, pasts, cnts = i32([p for t in trees for p in t]), i32(step.starts), i32(past), i32(counts)
    logits, probs, tokens, uniforms = map(dev, (j.logits, j.probs, j.tokens, j.uniforms))
    seen, positions = torch.zeros((T, 1), dtype=torch.int32, device=DEV), torch.zeros(T, dtype=torch.int32, device=DEV)
    path, lengths, chosen = (torch.zeros(s, dtype=torch.int32, device=DEV) for s in ((n, most), (n,), (n,)))
    out = torch.zeros((T, heads * dim), dtype=dtype, device=DEV)
    scratch = torch.zeros(max(1, ops.attention_tree_scratch_floats(T, n, most, heads, kv_heads, dim, stride * 64, dtype)), device=DEV)
    words = torch.zeros(max(1, ops.verify_drafts_scratch_words(n, T, vocab, True)), dtype=torch.int32, device=DEV)

    def run():
        ops.draft_tree(parents, starts, pasts, cnts, seen, positions, most)
        ops.attention_tree(q, k, v, out, starts, pasts, cnts, seen, positions, table, most, heads, kv_heads, dim, 0, step.scale, scratch=scratch)
        ops.verify_drafts(logits, vocab, tokens, parents, starts, cnts, uniforms, 1.0, path, lengths, chosen, most, probs=probs, scratch=words)
        ops.cache_compact(k, table, pasts, path, lengths, v_pool=v)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for t in (seen, positions, path, lengths, chosen, out):
        t.zero_()
    k.copy_(dev(step.k))
    v.copy_(dev(step.v))
    graph.replay()
    torch.cuda.synchronize()
    want = [plain.verify(j.logits[step.starts[s]:step.starts[s + 1]], j.tokens[step.starts[s]:step.starts[s + 1]], trees[s],
                         j.uniforms[step.starts[s]:step.starts[s + 1]], 1.0, vocab, j.probs[step.starts[s]:step.starts[s + 1]]) for s in range(n)]
    assert [path[s, :int(lengths[s])].tolist() for s in range(n)] == [w[0] for w in want] and chosen.tolist() == [w[1] for w in want]
    assert any(len(w[0]) > 1 for w in want)
    step.seen = torch.cat([plain.bits(plain.ways(t)[0], 1) for t in trees])
    ref, size, slack = step.want()
    rel = slack[..., None] + ((1 + 2.0 ** -8) ** 2 - 1 if dtype == torch.bfloat16 else 2.0 ** -23)
    assert bool(((out.cpu().view(T, heads, dim).double() - ref).abs() <= rel * size).all())
    # the next token: its row behind the rows that stay
    k_ref, v_ref = step.k.clone()[None], step.v.clone()[None]
    for pool in (k_ref, v_ref):
        plain.compact(pool, step.table, past, [w[0] for w in want])
    last = [p + len(w[0]) for p, w in zip(past, want)]
    for pool, ref_pool in ((k, k_ref), (v, v_ref)):
        got = pool.cpu()
        for s in range(n):
            for r in range(last[s]):
                page, at = step.place(s, r)
                assert torch.equal(got[page, :, at], ref_pool[0, page, :, at])
