"""What a cache of bounded size keeps: the policy's checks, the bookkeeping of pages, the command line (no GPU)."""

import random

import pytest

from sleuth_b200.cache.book import CacheBook, pages_for
from sleuth_b200.cache.keep import KeepPolicy
from sleuth_b200.engine.generate import plan_batches
from test_cache_book import invariants


def test_policy_checks():
    p = KeepPolicy(budget=100)
    assert (p.first, p.latest, p.most_rows) == (4, 50, 612)
    assert KeepPolicy(budget=5).latest == 1 and KeepPolicy(budget=9).latest == 4
    assert KeepPolicy(window=8, first=0).window == 8
    for kw in (dict(), dict(budget=4, window=4), dict(budget=-1), dict(budget=1.5), dict(window=True), dict(budget=8, first=9, recent=0),
               dict(budget=8, first=4, recent=5), dict(window=8, recent=2), dict(budget=8, portion=0), dict(budget=8, recent=-1)):
        with pytest.raises(ValueError):
            KeepPolicy(**kw)


def test_first_pages_stay_while_those_between_come_back():
    book = CacheBook([100], n_pages=40, max_slots=3, stride=20, firsts=[70])
    a, b = book.open(2)
    for n in (1, 64, 150, 300, 301, 640, 1280):
        need = book.pages_needed([a], [n])
        free = book.groups[0].pool.free
        book.grow([a], [n])
        assert free - book.groups[0].pool.free == need[0]
        book.commit([a], [n])
        row = book.groups[0].table[a]
        visible = [i for i in range(pages_for(n)) if i < 2 or 64 * i + 63 > n - 100]      # of queries from row n on
        assert [i for i in range(20) if row[i] >= 0] == visible
        assert book.seen[a] == book.lengths[a] == n
        invariants(book)
    book.close([a, b])
    invariants(book)


def test_peak_of_a_window_with_first_pages_is_what_the_steps_take():
    rng = random.Random(3)
    for _ in range(200):
        window, first = rng.randint(1, 300), rng.randint(0, 200)
        plan, n = [], 0
        while n < 1500:
            n += rng.randint(1, 400)
            plan.append(([0], [min(n, 1600)]))
        book = CacheBook([window], n_pages=60, max_slots=1, stride=25, firsts=[first])
        book.open(1)
        peak, = book.peak_pages_needed(plan)
        most = 0
        for slots, lens in plan:
            book.grow(slots, lens)
            most = max(most, book.pages_in_use()[0])
            book.commit(slots, lens)
            invariants(book)
        assert peak == most


def test_budget_bounds_rows_and_gives_pages_back():
    rng = random.Random(4)
    for _ in range(100):
        budget, portion = rng.randint(1, 300), rng.randint(1, 200)
        book = CacheBook([0], n_pages=2 * pages_for(budget + portion), max_slots=2, stride=pages_for(budget + portion), budget=budget)
        slots = book.open(2)
        seen = [0, 0]
        for _ in range(12):
            take = [rng.randint(1, portion) for _ in slots]
            lens = [int(book.lengths[s]) + t for s, t in zip(slots, take)]
            need = book.pages_needed(slots, lens)
            free = book.groups[0].pool.free
            assert book.peak_pages_needed([(slots, lens)]) == need
            book.grow(slots, lens)
            assert free - book.groups[0].pool.free == need[0]
            book.commit(slots, lens)
            invariants(book)
            for i, (s, t) in enumerate(zip(slots, take)):
                seen[i] += t
                assert book.seen[s] == seen[i] and book.lengths[s] == min(lens[i], budget)
                row = book.groups[0].table[s]
                assert (row[:pages_for(int(book.lengths[s]))] >= 0).all() and (row[pages_for(int(book.lengths[s])):] < 0).all()
        book.close(slots)
        assert book.pages_in_use() == [0] and not book.seen.any()


def test_batches_are_planned_by_the_rows_that_are_kept():
    assert plan_batches([5000, 5000, 5000], 100, 8192, 24, 8) == [[0], [1], [2]]
    assert plan_batches([5000, 5000, 5000], 100, 8192, 24, 8, max_rows=512) == [[0, 1, 2]]


def test_command_line_offers_the_policy():
    from sleuth_b200.cli import build_parser
    a = build_parser().parse_args(["generate", "m", "--keep-budget", "512", "--keep-first", "2", "--keep-recent", "100"])
    assert (a.keep_budget, a.keep_first, a.keep_recent, a.keep_window) == (512, 2, 100, 0)
    b = build_parser().parse_args(["generate", "m"])
    assert (b.keep_budget, b.keep_window) == (0, 0)


def test_designs_that_it_is_not_built_for_are_refused():
    from types import SimpleNamespace as N

    from sleuth_b200.engine.engine import _check_keep
    entry = lambda c, borrow=-1: N(cache=c, borrow=borrow)  # noqa: E731
    layer = lambda kind: N(mixer=N(kind=kind))  # noqa: E731
    good = N(layers=[layer("gqa_attention")], schedule=[entry(0), entry(1)])
    _check_keep(None, N(layers=[layer("retention")], schedule=[]))
    _check_keep(KeepPolicy(window=5), good)
    with pytest.raises(ValueError):
        _check_keep(KeepPolicy(window=5), N(layers=[layer("gqa_attention"), layer("retention")], schedule=[entry(0)]))
    with pytest.raises(ValueError):
        _check_keep(KeepPolicy(window=5), N(layers=[layer("gqa_attention")], schedule=[entry(0), entry(0)]))
    with pytest.raises(ValueError):
        _check_keep(KeepPolicy(window=5), N(layers=[layer("gqa_attention")], schedule=[entry(0), entry(1, borrow=0)]))
    with pytest.raises(TypeError):
        _check_keep(dict(window=5), good)


def test_plain_eviction_keeps_what_it_should():
    from plain import kept_plain
    source, at = kept_plain.evict([5, 1, 1, 9, 0, 3], [0, 1, 2, 3, 4, 5], 6, 6, 6, 4, 1, 1)
    assert source == [0, 1, 5, 3] and at == [0, 1, 5, 3]      # rows 2 and 4 go (1 ties with 2: the lower stays), row 5 fills the first place
    assert kept_plain.evict([1, 2], [0, 1], 2, 2, 2, 4, 1, 1)[0] == [0, 1]
