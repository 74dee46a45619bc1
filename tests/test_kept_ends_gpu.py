"""The operators of a cache of bounded size at the ends of their arguments' ranges."""

import math

import pytest
import torch

from plain import kept_plain as plain
from test_kept_gpu import DEV, Step

pytestmark = pytest.mark.gpu

MOST = 2 ** 31 - 1
KINDS = [(torch.float32, 6, 3, 24), (torch.float32, 8, 2, 64), (torch.bfloat16, 4, 2, 64), (torch.bfloat16, 16, 8, 128), (torch.bfloat16, 6, 2, 128)]
KIND_IDS = [f"{str(d)[6:]}-{h}-{k}-{e}" for d, h, k, e in KINDS]


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("window,first", [(MOST, 4), (MOST - 150, 0), (MOST, MOST), (5, MOST), (40, MOST - 62), (MOST - 1, MOST - 63)])
@pytest.mark.parametrize("count", [1, 3, 200])
def test_largest_windows_and_first_rows(dtype, heads, kv_heads, dim, window, first, count):
    """A program says "no limit" with the largest number there is."""
    Step(dtype, heads, kv_heads, dim, [0, 70, 131], [count, 1, count], window, first, seed=11).check(weights=True, lse=True, promise=count != 3)


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("counts", [[1, 1], [3, 2], [150, 70]])
def test_largest_promise_of_new_tokens(dtype, heads, kv_heads, dim, counts):
    """``max_count`` and ``max_keys`` are upper limits: the largest numbers there are say nothing, and cost no result."""
    from sleuth_b200.kernels import ops
    step = Step(dtype, heads, kv_heads, dim, [90, 3], counts, 60, 5, seed=12)
    t = step.tensors()
    out = torch.empty((step.T, heads * dim), dtype=dtype, device=DEV)
    w = step.weights.to(DEV)
    floats = ops.attention_kept_scratch_floats(step.T, 2, MOST, heads, kv_heads, dim, 64 * step.stride, dtype, weights=True)
    ops.attention_kept(t["q"], t["k"], t["v"], out, t["seq_start"], t["past"], t["counts"], t["table"], MOST, heads, kv_heads, dim, 60, 5, step.scale,
                       scratch=torch.empty(max(1, floats), device=DEV), max_keys=MOST, weights=w)
    want, _, _, want_w = plain.attention(step.q, step.k, step.v, step.seq_start, step.past, step.counts, step.table, heads, kv_heads, 60, 5, step.scale, step.weights)
    # (the same bounds as in the tests of the sizes in between)
    _, _, size, _ = plain.attention(step.q, step.k, step.v, step.seq_start, step.past, step.counts, step.table, heads, kv_heads, 60, 5, step.scale)
    rel = 2.0 ** -7 if dtype == torch.bfloat16 else 5e-5
    assert bool(((out.cpu().view(want.shape).double() - want).abs() <= rel * size + 1e-12).all())
    for s, (p, c) in enumerate(zip(step.past, step.counts)):
        assert bool(((w[s, :, :p + c].cpu().double() - want_w[s, :, :p + c]).abs() <= 5e-5 * want_w[s, :, :p + c].abs() + 1e-7).all())


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("past,counts", [([40, 700, 9], [1, 0, 1]), ([0, 130], [0, 1]), ([70, 300, 0, 64], [3, 0, 0, 2]), ([500, 20], [0, 150]),
                                         ([3000, 10, 65], [0, 300, 0])])
@pytest.mark.parametrize("window,first", [(0, 0), (50, 5)])
def test_sequences_without_new_tokens_keep_what_they_gathered(dtype, heads, kv_heads, dim, past, counts, window, first):
    step = Step(dtype, heads, kv_heads, dim, past, counts, window, first, seed=13)
    for slots in (None, [len(past) - i for i in range(len(past))]):
        for in_place in (True, False):
            _, _, got = step.run(weights=True, in_place=in_place, slots=slots)
            for s, (p, c) in enumerate(zip(past, counts)):
                if c == 0:
                    assert torch.equal(got[s, :, :p], step.weights[s, :, :p])
                    rest = step.weights[s, :, p:] if in_place else torch.full_like(got[s, :, p:], -5.0)
                    assert torch.equal(got[s, :, p:], rest)


@pytest.mark.parametrize("slots", [None, [2, 0]])
def test_a_step_without_any_token_keeps_what_was_gathered(slots):
    from sleuth_b200.kernels import ops
    past, K, cap = [200, 3], 2, 5 * 64
    w = torch.rand((3, K, cap), device=DEV)
    target = torch.full_like(w, -5.0)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    pool = torch.zeros((10, K, 64, 64), dtype=torch.bfloat16, device=DEV)
    q, out = torch.empty((0, 4, 64), dtype=torch.bfloat16, device=DEV), torch.empty((0, 256), dtype=torch.bfloat16, device=DEV)
    ops.attention_kept(q, pool, pool, out, i32([0, 0, 0]), i32(past), i32([0, 0]), torch.zeros((2, 5), dtype=torch.int32, device=DEV), 0, 4, K, 64, 0, 0, 0.1,
                       weights=w, weights_out=target, slots=None if slots is None else i32(slots))
    want = torch.full_like(w, -5.0)
    for s, p in enumerate(past):
        at = s if slots is None else slots[s]
        want[at, :, :p] = w[at, :, :p]
    assert torch.equal(target, want)


def _evict_call(cap, stride=4, **kw):
    from sleuth_b200.kernels import ops
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    pool = torch.zeros((stride, 2, 64, 16), device=DEV)
    a = dict(weights=torch.rand((1, 2, cap), device=DEV), positions=torch.zeros((1, 2, cap), dtype=torch.int32, device=DEV), k_pool=pool, v_pool=pool.clone(),
             block_table=torch.arange(stride, dtype=torch.int32, device=DEV).view(1, -1), past=i32([50]), lengths=i32([90]), seen=i32([90]), budget=60, first=2,
             recent=3, scratch=torch.empty(10000, dtype=torch.int32, device=DEV))
    a.update(kw)
    ops.cache_evict(**a)


def test_evictions_refuse_weights_that_are_shorter_than_the_cache():
    """A row that weights and positions have no place for cannot be ranked, and no position behind it can be told."""
    _evict_call(256)
    _evict_call(100, max_length=100)
    _evict_call(300, max_length=5000)
    for cap, kw in ((255, {}), (80, {}), (99, dict(max_length=100)), (80, dict(max_length=90)), (255, dict(max_length=5000))):
        with pytest.raises(ValueError):
            _evict_call(cap, **kw)


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("past,counts,token", [([30, 200], [1, 1], 0), ([30, 200], [5, 3], 6), ([0, 90], [200, 70], 60), ([64, 10], [150, 140], 149)])
@pytest.mark.parametrize("window,first", [(0, 0), (40, 6)])
def test_a_query_that_is_not_a_number_spoils_only_what_it_sees(dtype, heads, kv_heads, dim, past, counts, token, window, first):
    step = Step(dtype, heads, kv_heads, dim, past, counts, window, first, seed=14, hole=False)
    step.q[token, heads - 1, 0] = math.nan
    out, lse, got = step.run(weights=True, lse=True)
    want, want_lse, size, want_w = plain.attention(step.q, step.k, step.v, step.seq_start, past, counts, step.table, heads, kv_heads, window, first, step.scale,
                                                   step.weights)
    # (the same bounds as in the tests of finite queries)
    rel = 2.0 ** -7 if dtype == torch.bfloat16 else 5e-5
    assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(torch.isnan(lse), torch.isnan(want_lse))
    assert bool(((out - want).abs() <= rel * size + 1e-12)[~torch.isnan(want)].all())
    for s, (p, c) in enumerate(zip(past, counts)):
        a, b = got[s, :, :p + c].double(), want_w[s, :, :p + c]
        assert torch.equal(torch.isnan(a), torch.isnan(b)), (s, torch.isnan(a).sum(-1).tolist(), torch.isnan(b).sum(-1).tolist())
        assert bool(((a - b).abs() <= 5e-5 * b.abs() + 1e-7)[~torch.isnan(b)].all())


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", [KINDS[0], KINDS[1], KINDS[4]], ids=[KIND_IDS[0], KIND_IDS[1], KIND_IDS[4]])
@pytest.mark.parametrize("window,first", [(1, 0), (63, 1), (64, 64), (65, 3), (300, 130)])
@pytest.mark.parametrize("count", [1, 4, 23, 70])
def test_short_windows_on_a_long_table(dtype, heads, kv_heads, dim, window, first, count):
    """Shares of the keys go by what a tile sees, not by the table's length (no promise of a length is made)."""
    step = Step(dtype, heads, kv_heads, dim, [1500, 0, 64], [count, 1, max(1, count - 1)], window, first, seed=15)
    step.check(weights=True, lse=True, promise=False)


def test_an_engine_with_the_largest_policies(tmp_path):
    """A budget, a portion, a window or first tokens without a limit are the whole cache."""
    import numpy as np

    import sleuth_b200 as sb
    import tiny
    cfg = tiny.CONFIGS["D"]
    sb.write_random_model(tmp_path, cfg, seed=9, dtype=torch.float32)
    prompts = [np.random.default_rng(1).integers(0, cfg["vocab_size"], n).tolist() for n in (150, 9)]
    rows = []
    for keep in (None, sb.KeepPolicy(budget=MOST, portion=MOST), sb.KeepPolicy(budget=MOST, first=MOST, recent=0, portion=40), sb.KeepPolicy(window=MOST, first=4),
                 sb.KeepPolicy(window=7, first=MOST)):
        engine = sb.load(tmp_path, dtype="fp32", max_seq_len=300, device="cuda:0", keep=keep)
        assert engine.cache.stride == 5
        slots = engine.open(2)
        out = [engine.step([(s, p, (len(p) - 1,)) for s, p in zip(slots, prompts)]).cpu()]
        for turn in ([3], [4, 5, 6], [7]):
            out.append(engine.step([(s, turn, (len(turn) - 1,)) for s in slots]).cpu().clone())
        rows.append(torch.cat(out))
        engine.stepper.check_status()
    for r in rows[1:]:      # (sums of at most a few hundred terms in another order)
        assert float((r - rows[0]).abs().max()) <= 1e-5 * float(rows[0].abs().max())


def test_the_command_line_generates_beyond_its_budget(tmp_path, capsys):
    import sleuth_b200 as sb
    import tiny
    from sleuth_b200.cli import main
    sb.write_random_model(tmp_path, tiny.CONFIGS["D"], seed=9, dtype=torch.float32)
    assert main(["generate", str(tmp_path), "--prompt-ids", "1 2 3; 7 8", "--max-new-tokens", "150", "--temperature", "0", "--max-seq-len", "300",
                 "--keep-budget", "64", "--samples", "2"]) == 0
    lines = [[int(t) for t in x.split()] for x in capsys.readouterr().out.splitlines() if x and x[0].isdigit()]
    assert len(lines) == 4 and lines[0] == lines[2] and lines[1] == lines[3] and all(lines)
