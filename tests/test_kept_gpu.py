"""Attention over a cache of bounded size, the weights that its rows gather, and eviction, against the formulas in 64 bits."""

import math

import pytest
import torch

from plain import kept_plain as plain

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


class Step:
    """A step with its cache: pools whose unused rows hold NaN, pages in no order, pages that no query sees taken out of the table."""

    def __init__(self, dtype, heads, kv_heads, dim, past, counts, window=0, first=0, seed=0, sharp=1.5, hole=True):
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.heads, self.kv_heads, self.dim = dtype, heads, kv_heads, dim
        self.past, self.counts, self.window, self.first = list(past), list(counts), window, first
        n = len(past)
        longest = max(p + c for p, c in zip(past, counts))
        self.stride = max(1, -(-longest // 64)) + 1
        pages = n * self.stride + 2
        self.k = torch.full((pages, kv_heads, 64, dim), math.nan, dtype=dtype)
        self.v = torch.full((pages, kv_heads, 64, dim), math.nan, dtype=dtype)
        order = torch.randperm(pages, generator=g)
        self.table = torch.full((n, self.stride), -1, dtype=torch.int32)
        at = 0
        for s, (p, c) in enumerate(zip(past, counts)):
            for i in range(-(-(p + c) // 64)):
                page = int(order[at])
                at += 1
                rows = min(64, p + c - 64 * i)
                self.k[page, :, :rows] = torch.randn((kv_heads, rows, dim), generator=g).to(dtype)
                self.v[page, :, :rows] = torch.randn((kv_heads, rows, dim), generator=g).to(dtype)
                hidden = window and c and 64 * i >= first and 64 * i + 63 <= p - window
                if hidden:          # no query of the step sees it: a cache gives such pages back
                    self.k[page] = math.nan
                    self.v[page] = math.nan
                if not (hidden and hole):
                    self.table[s, i] = page
            if window and c:        # rows of pages that are held, but that no query sees
                for j in range(first, max(first, p - window + 1)):
                    page = int(self.table[s, j // 64])
                    if page >= 0:
                        self.k[page, :, j % 64] = math.inf
                        self.v[page, :, j % 64] = math.nan
        starts = [0]
        for c in counts:
            starts.append(starts[-1] + c)
        self.T = starts[-1]
        self.seq_start = torch.tensor(starts, dtype=torch.int32)
        self.q = (sharp * torch.randn((self.T, heads, dim), generator=g)).to(dtype)
        self.scale = dim ** -0.5
        self.weights = torch.rand((n, kv_heads, self.stride * 64), generator=g)
        self.max_keys = longest

    def tensors(self):
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
        return dict(q=self.q.to(DEV), k=self.k.to(DEV), v=self.v.to(DEV), table=self.table.to(DEV), seq_start=self.seq_start.to(DEV),
                    past=i32(self.past), counts=i32(self.counts))

    def run(self, weights=False, lse=False, in_place=True, slots=None, promise=True, stream=None):
        from sleuth_b200.kernels import ops
        t = self.tensors()
        n = len(self.past)
        floats = ops.attention_kept_scratch_floats(self.T, n, max(self.counts), self.heads, self.kv_heads, self.dim,
                                                   self.max_keys if promise else self.stride * 64, self.dtype, weights=weights)
        scratch = torch.full((max(floats, 1),), math.nan, device=DEV)
        out = torch.full((self.T, self.heads * self.dim), 7.0, dtype=self.dtype, device=DEV)
        lse_t = torch.full((self.T, self.heads), 7.0, device=DEV) if lse else None
        kw = {}
        if weights:
            w = self.weights
            if slots is not None:
                w = torch.full((max(slots) + 1, *self.weights.shape[1:]), -3.0)
                w[slots] = self.weights
            w = w.to(DEV).contiguous()
            target = w if in_place else torch.full_like(w, -5.0)
            kw = dict(weights=w, weights_out=None if in_place else target)
            if slots is not None:
                kw["slots"] = torch.tensor(slots, dtype=torch.int32, device=DEV)
        torch.cuda.synchronize()
        ops.attention_kept(t["q"], t["k"], t["v"], out, t["seq_start"], t["past"], t["counts"], t["table"], max(self.counts), self.heads,
                           self.kv_heads, self.dim, self.window, self.first, self.scale, scratch=scratch,
                           max_keys=self.max_keys if promise else 0, lse=lse_t, stream=stream, **kw)
        torch.cuda.synchronize()
        assert ops.tc_status(out.device) is None or int(ops.tc_status(out.device)) == 0
        got_w = None
        if weights:
            got_w = target.cpu()
            got_w = got_w[slots] if slots is not None else got_w
        return out.cpu().view(self.T, self.heads, self.dim).double(), None if lse_t is None else lse_t.cpu().double(), got_w

    def check(self, weights=False, lse=False, **kw):
        out, got_lse, got_w = self.run(weights, lse, **kw)
        want, want_lse, size, want_w = plain.attention(self.q, self.k, self.v, self.seq_start, self.past, self.counts, self.table, self.heads,
                                                       self.kv_heads, self.window, self.first, self.scale, self.weights if weights else None)
        # float32: a score is a sum of up to 256 products of size up to 30, so it is off by a few 1e-6 at most in either order, and a
        # weight by that share; the weighted sum adds one rounding per key in the worst case, a few in fact. bfloat16: the
        # weights and the result are rounded once each, half of 2^-8 relative, and the scores' sums as in float32
        rel = 2.0 ** -7 if self.dtype == torch.bfloat16 else 5e-5
        err = (out - want).abs()
        assert torch.isfinite(out).all()
        assert bool((err <= rel * size + 1e-12).all()), float((err / (size + 1e-12)).max())
        if lse:
            assert bool(((got_lse - want_lse).abs() <= 5e-5 * (1 + want_lse.abs())).all())
        if weights:
            for s, (p, c) in enumerate(zip(self.past, self.counts)):
                if c == 0:
                    continue
                a, b = got_w[s, :, :p + c].double(), want_w[s, :, :p + c]
                assert bool(((a - b).abs() <= 5e-5 * b.abs() + 1e-7).all()), float((a - b).abs().max())
                if kw.get("in_place", True):         # rows behind the last are left alone
                    assert torch.equal(got_w[s, :, p + c:], self.weights[s, :, p + c:])


HEADS = [(torch.float32, 6, 3, 24), (torch.float32, 4, 4, 10), (torch.float32, 8, 2, 64), (torch.float32, 4, 2, 128), (torch.float32, 2, 1, 256),
         (torch.bfloat16, 4, 2, 64), (torch.bfloat16, 4, 1, 128), (torch.bfloat16, 6, 2, 128), (torch.bfloat16, 16, 1, 64),
         (torch.bfloat16, 3, 3, 96), (torch.bfloat16, 20, 1, 64)]
IDS = [f"{str(d)[6:]}-{h}-{k}-{e}" for d, h, k, e in HEADS]


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", HEADS, ids=IDS)
@pytest.mark.parametrize("window,first", [(0, 0), (1, 0), (1, 1), (37, 4), (64, 64), (150, 100), (4096, 4)])
def test_single_tokens(dtype, heads, kv_heads, dim, window, first):
    Step(dtype, heads, kv_heads, dim, [0, 1, 63, 64, 65, 200, 450], [1] * 7, window, first, seed=1).check(weights=True, lse=True)


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", HEADS, ids=IDS)
@pytest.mark.parametrize("window,first", [(0, 0), (2, 1), (50, 3), (100, 70)])
def test_few_tokens(dtype, heads, kv_heads, dim, window, first):
    Step(dtype, heads, kv_heads, dim, [0, 5, 62, 130, 300, 9], [3, 7, 2, 5, 6, 0], window, first, seed=2).check(weights=True, lse=True)


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", HEADS, ids=IDS)
@pytest.mark.parametrize("window,first", [(0, 0), (1, 1), (40, 4), (130, 200)])
def test_prompts_and_portions(dtype, heads, kv_heads, dim, window, first):
    Step(dtype, heads, kv_heads, dim, [0, 0, 70, 0, 333], [1, 150, 90, 0, 67], window, first, seed=3).check(weights=True, lse=True)


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", [HEADS[2], HEADS[5], HEADS[6]], ids=["float32", "bfloat16-64", "bfloat16-128"])
@pytest.mark.parametrize("count", [1, 4, 40, 200])
def test_without_promise_without_weights_apart_and_in_other_slots(dtype, heads, kv_heads, dim, count):
    step = Step(dtype, heads, kv_heads, dim, [100, 3, 260], [count] * 3, 90, 10, seed=4)
    step.check(promise=False)
    step.check(weights=True, in_place=False)
    step.check(weights=True, slots=[4, 0, 2])
    step.check(weights=True, promise=False, lse=True)


@pytest.mark.parametrize("dtype,dim", [(torch.float32, 24), (torch.float32, 64), (torch.bfloat16, 64), (torch.bfloat16, 128)])
@pytest.mark.parametrize("count", [1, 5, 130])
def test_lowest_scores_and_rows_without_weight(dtype, dim, count):
    """Scores far apart, keys of -inf that leave a row nothing, and one key that takes it all."""
    step = Step(dtype, 4, 2, dim, [10, 120], [count, count], 0, 0, seed=5, sharp=20.0)
    step.q[:, 0, :] = 0
    step.q[:, 0, 0] = 1.0          # head 0 looks at the first channel, and finds -inf everywhere in kv head 0
    step.k[:, 0, :, 0] = -math.inf
    step.q[:, 1, 0] = 0.0          # 0 * -inf: the other head of the group sees NaN; it is left out below
    t, got_lse, got_w = step.run(weights=True, lse=True)
    assert bool((t[:, 0] == 0).all()) and bool((got_lse[:, 0] == -math.inf).all())
    assert bool(torch.isnan(t[:, 1]).all())
    want, want_lse, size, _ = plain.attention(step.q[:, 2:], step.k[:, 1:], step.v[:, 1:], step.seq_start, step.past, step.counts, step.table, 2, 1,
                                              0, 0, step.scale)
    # scores up to some hundred: a sum of them is off by 1e-5 relative at most, so a weight by a few 1e-3 (float32) as an upper bound
    rel = 2.0 ** -6 if dtype == torch.bfloat16 else 5e-3
    assert bool(((t[:, 2:] - want).abs() <= rel * size + 1e-12).all())


def test_on_another_stream_and_twice_the_same_bits():
    step = Step(torch.bfloat16, 8, 2, 128, [700, 3, 64], [1, 1, 1], 500, 4, seed=6)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        a = step.run(weights=True, stream=s.cuda_stream)
    b = step.run(weights=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2])
    step = Step(torch.bfloat16, 8, 2, 128, [70, 0], [140, 300], 100, 4, seed=6)
    a, b = step.run(weights=True), step.run(weights=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2])


def test_rows_far_into_a_large_pool():
    """Offsets beyond 2^31 elements: a pool of 5 GB whose last pages are the sequence's."""
    from sleuth_b200.kernels import ops
    pages, K, dim = 150000, 2, 128
    k = torch.zeros((pages, K, 64, dim), dtype=torch.bfloat16, device=DEV)
    g = torch.Generator().manual_seed(8)
    small = Step(torch.bfloat16, 4, K, dim, [190], [1], 100, 10, seed=9, hole=False)
    t = small.tensors()
    held = small.table[0][small.table[0] >= 0]
    far = torch.randperm(200, generator=g)[:held.numel()] + pages - 200
    v = torch.zeros_like(k)
    k[far.to(DEV)], v[far.to(DEV)] = t["k"][held.long().to(DEV)], t["v"][held.long().to(DEV)]
    table = torch.full((1, small.stride), -1, dtype=torch.int32, device=DEV)
    table[0, :held.numel()] = far.to(torch.int32).to(DEV)
    for count in (1, 40, 140):
        step = Step(torch.bfloat16, 4, K, dim, [191 - count], [count], 100, 10, seed=9, hole=False)
        q = step.q.to(DEV)
        outs = []
        for kk, vv, tt in ((t["k"], t["v"], t["table"]), (k, v, table)):
            out = torch.empty((count, 4 * dim), dtype=torch.bfloat16, device=DEV)
            w = torch.zeros((1, K, small.stride * 64), device=DEV)
            floats = ops.attention_kept_scratch_floats(count, 1, count, 4, K, dim, 191, torch.bfloat16, weights=True)
            tables = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0, count], [191 - count], [count])]
            kk, vv = torch.nan_to_num(kk, 0.0, 0.0, 0.0) if kk is t["k"] else kk, torch.nan_to_num(vv, 0.0, 0.0, 0.0) if vv is t["v"] else vv
            if kk is k:
                k[far.to(DEV)] = torch.nan_to_num(k[far.to(DEV)], 0.0, 0.0, 0.0)
                v[far.to(DEV)] = torch.nan_to_num(v[far.to(DEV)], 0.0, 0.0, 0.0)
            ops.attention_kept(q, kk, vv, out, *tables, tt, count, 4, K, dim, 100, 10, step.scale,
                               scratch=torch.empty(max(floats, 1), device=DEV), max_keys=191, weights=w)
            outs.append((out.cpu(), w.cpu()))
        assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


# ------------------------------------------------------------------ eviction ----

def _evict_case(dtype, kv_heads, dim, lengths, past, budget, first, recent, seed=0, gone=0, kind="plain", in_place=True, slots=None, promise=True):
    from sleuth_b200.kernels import ops
    g = torch.Generator().manual_seed(seed)
    n, stride = len(lengths), max(1, -(-max(lengths) // 64)) + 1
    cap = stride * 64 + 5
    pages = n * stride + 1
    k = torch.randn((pages, kv_heads, 64, dim), generator=g).to(dtype)
    v = torch.randn((pages, kv_heads, 64, dim), generator=g).to(dtype)
    table = torch.randperm(pages, generator=g)[:n * stride].view(n, stride).to(torch.int32)
    w = torch.rand((n, kv_heads, cap), generator=g)
    if kind == "ties":
        w = (w * 4).floor() / 4 - 0.25
        w[w == 0] = -0.0
        w[:, :, ::7] = 0.0
    elif kind == "same":
        w[:] = 0.5
    elif kind == "odd":
        pick = torch.rand(w.shape, generator=g)
        w[pick < 0.2] = math.nan
        w[(pick > 0.2) & (pick < 0.3)] = math.inf
        w[(pick > 0.3) & (pick < 0.4)] = -math.inf
        w[(pick > 0.4) & (pick < 0.5)] = 1e-42
    seen = [m + gone for m in lengths]
    pos = torch.full((n, kv_heads, cap), -9, dtype=torch.int32)
    for s in range(n):
        for h in range(kv_heads):
            fresh = lengths[s] - past[s]
            pos[s, h, :past[s]] = torch.randperm(seen[s] - fresh, generator=g)[:past[s]].to(torch.int32)
    slot_of = list(range(n)) if slots is None else slots
    W = torch.full((max(slot_of) + 1, kv_heads, cap), -3.0)
    P = torch.full((max(slot_of) + 1, kv_heads, cap), -3, dtype=torch.int32)
    W[slot_of], P[slot_of] = w, pos
    dk, dv, dW, dP = k.to(DEV), v.to(DEV), W.to(DEV), P.to(DEV)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    outW, outP = (dW, dP) if in_place else (torch.full_like(dW, -7.0), torch.full_like(dP, -7))
    longest = max(lengths) if promise else 0
    words = ops.cache_evict_scratch_words(n, kv_heads, budget, longest or stride * 64)
    ops.cache_evict(dW, dP, dk, dv, table.to(DEV), i32(past), i32(lengths), i32(seen), budget, first, recent, weights_out=None if in_place else outW,
                    positions_out=None if in_place else outP, slots=None if slots is None else i32(slots),
                    scratch=torch.full((max(words, 1),), -1, dtype=torch.int32, device=DEV), max_length=longest)
    torch.cuda.synchronize()
    outW, outP, dk, dv = outW.cpu(), outP.cpu(), dk.cpu(), dv.cpu()
    want_k, want_v = k.clone(), v.clone()
    for s in range(n):
        for h in range(kv_heads):
            source, at = plain.evict(w[s, h], pos[s, h], past[s], lengths[s], seen[s], budget, first, recent)
            left = len(source)
            src = torch.tensor(source, dtype=torch.long)
            got = outW[slot_of[s], h, :left]
            assert torch.equal(got.view(torch.int32), w[s, h][src].contiguous().view(torch.int32))
            assert outP[slot_of[s], h, :left].tolist() == at
            rest = (W[slot_of[s], h, left:], P[slot_of[s], h, left:]) if in_place else (torch.full_like(outW[0, 0, left:], -7.0), torch.full_like(outP[0, 0, left:], -7))
            if lengths[s] > left or not in_place:
                assert torch.equal(outW[slot_of[s], h, left:].view(torch.int32), rest[0].contiguous().view(torch.int32))
            to = torch.arange(left)
            pg = table[s].long()
            want_k[pg[to // 64], h, to % 64] = k[pg[src // 64], h, src % 64]
            want_v[pg[to // 64], h, to % 64] = v[pg[src // 64], h, src % 64]
    assert torch.equal(dk, want_k) and torch.equal(dv, want_v)


@pytest.mark.parametrize("kind", ["plain", "ties", "same", "odd"])
@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.float32, 24), (torch.bfloat16, 10)])
def test_evict_a_row_a_step(kind, dtype, dim):
    for seed, (budget, first, recent) in enumerate([(1, 0, 0), (1, 0, 1), (1, 1, 0), (7, 2, 3), (64, 4, 16), (200, 0, 200), (200, 4, 50), (1500, 4, 100)]):
        _evict_case(dtype, 3, dim, [budget + 1, max(1, budget), budget + 1], [budget, max(0, budget - 1), budget], budget, first, recent, seed=seed,
                    gone=40, kind=kind)


@pytest.mark.parametrize("kind", ["plain", "ties", "same", "odd"])
@pytest.mark.parametrize("in_place", [True, False])
def test_evict_after_prompts(kind, in_place):
    _evict_case(torch.bfloat16, 2, 64, [1, 63, 500, 3000, 1025], [0] * 5, 100, 4, 20, seed=3, kind=kind, in_place=in_place)
    _evict_case(torch.bfloat16, 2, 128, [900, 4100], [500, 100], 512, 0, 64, seed=4, kind=kind, gone=77, in_place=in_place)
    _evict_case(torch.float32, 1, 16, [300, 130, 20], [128, 128, 19], 129, 3, 0, seed=5, kind=kind, gone=5, in_place=in_place, slots=[2, 0, 5])
    _evict_case(torch.float32, 2, 16, [300, 260], [256, 256], 256, 1, 3, seed=6, kind=kind, gone=5, in_place=in_place, promise=False)


@pytest.mark.parametrize("kind", ["plain", "ties", "same", "odd"])
@pytest.mark.parametrize("in_place", [True, False])
def test_evict_around_and_beyond_the_rows_a_block_reads_at_once(kind, in_place):
    _evict_case(torch.bfloat16, 2, 16, [8191, 8192, 8193, 20011], [8000, 8192, 0, 16385], 700, 5, 300, seed=9, kind=kind, gone=33, in_place=in_place)
    _evict_case(torch.bfloat16, 1, 16, [2047, 2048, 33], [2000, 0, 33], 1500, 0, 1500, seed=10, kind=kind, in_place=in_place)


def test_evict_more_rows_than_shared_memory_holds():
    _evict_case(torch.bfloat16, 1, 16, [50001, 100], [50000, 100], 50000, 4, 100, seed=7, kind="ties", gone=9)
    _evict_case(torch.bfloat16, 1, 16, [60000], [100], 3000, 4, 100, seed=8, kind="plain", gone=9)


# ------------------------------------------------------------------ refusals ----

def test_refusals():
    from sleuth_b200.kernels import ops
    step = Step(torch.bfloat16, 4, 2, 64, [10], [1], seed=1)
    t = step.tensors()
    out = torch.empty((1, 256), dtype=torch.bfloat16, device=DEV)
    w = torch.zeros((1, 2, step.stride * 64), device=DEV)

    def call(**kw):
        a = dict(q=t["q"], k_pool=t["k"], v_pool=t["v"], out=out, seq_start=t["seq_start"], past=t["past"], counts=t["counts"], block_table=t["table"],
                 max_count=1, heads=4, kv_heads=2, head_dim=64, window=0, first=0, scale=0.1, scratch=torch.empty(100000, device=DEV))
        a.update(kw)
        ops.attention_kept(**a)

    call()
    for kw in (dict(window=-1), dict(first=-1), dict(q=t["q"].float()), dict(q=t["q"].cpu()), dict(out=out[:, :128]), dict(block_table=t["table"].long()),
               dict(heads=5), dict(k_pool=t["k"][:, :1]), dict(past=t["past"].float()), dict(counts=t["counts"][:0]), dict(lse=torch.empty(4, device=DEV)),
               dict(weights_out=w), dict(weights=w[:, :1].contiguous()), dict(weights=w[:, :, :5].contiguous()), dict(weights=w.double()),
               dict(weights=w, weights_out=w[:, :, :-1].contiguous()), dict(slots=t["past"].long()), dict(v_pool=t["v"].transpose(1, 2))):
        with pytest.raises(ValueError):
            call(**kw)
    with pytest.raises(RuntimeError):       # (float32 keeps the denominators in scratch, whatever the step)
        call(weights=w, scratch=None, q=t["q"].float(), out=out.float(), k_pool=t["k"].float(), v_pool=t["v"].float())
    with pytest.raises(RuntimeError):
        call(q=t["q"][:, :3].contiguous(), heads=3, out=out[:, :192].contiguous())
    pos = torch.zeros((1, 2, step.stride * 64), dtype=torch.int32, device=DEV)

    def evict(**kw):
        a = dict(weights=w, positions=pos, k_pool=t["k"], v_pool=t["v"], block_table=t["table"], past=t["past"], lengths=t["counts"], seen=t["past"],
                 budget=8, first=2, recent=2, scratch=torch.empty(10000, dtype=torch.int32, device=DEV))
        a.update(kw)
        ops.cache_evict(**a)

    evict()
    for kw in (dict(budget=0), dict(first=5, recent=4), dict(first=-1), dict(recent=-1), dict(weights=w.half()), dict(positions=pos.long()),
               dict(positions=pos[:, :, :-1].contiguous()), dict(k_pool=t["k"].float()), dict(lengths=t["counts"].long()), dict(weights_out=w[:, :1].contiguous()),
               dict(seen=t["past"][:0]), dict(scratch=torch.empty(10, device=DEV)), dict(weights=w.cpu())):
        with pytest.raises(ValueError):
            evict(**kw)
    with pytest.raises(RuntimeError):
        evict(scratch=None, budget=60, max_length=128)
