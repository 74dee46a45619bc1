"""Steps of drafted tokens that nobody accepts: slots that were closed, pages that were taken, drafts that were counted. No GPU."""

import types

import pytest
import torch

from sleuth_b200.cache.book import CacheBook, CacheMisuse
from sleuth_b200.engine.engine import Engine
from sleuth_b200.engine.generate import generate_batches
from sleuth_b200.engine.stepper import Stepper
from sleuth_b200.sampling import DraftPolicy, SamplingConfig

from test_drafts_loop import Drafting


def bare_engine(book):
    """The slots' book-keeping of an engine, without a model or a device."""
    engine, stepper = object.__new__(Engine), object.__new__(Stepper)
    stepper._drafted, stepper.cache = {}, types.SimpleNamespace(book=book, pools=[], open=book.open, close=book.close)
    engine.stepper, engine.cache = stepper, stepper.cache
    return engine


def drafted(engine, slot, count):
    """As ``step_tree`` leaves a slot."""
    book = engine.cache.book
    past = int(book.lengths[slot])
    book.grow([slot], [past + count])
    engine.stepper._drafted[slot] = (past, count)


def whole(book):
    held = [sorted(p for row in g.table for p in row if p >= 0) for g in book.groups]
    return all(sorted(h + list(g.pool._free)) == list(range(g.pool.n_pages)) for h, g in zip(held, book.groups))


def test_a_closed_slot_accepts_nothing():
    book = CacheBook([0, 40], 8, 2, stride=4)
    engine = bare_engine(book)
    a, = engine.open(1)
    drafted(engine, a, 60)
    engine.close([a])
    with pytest.raises(ValueError, match="accept"):
        engine.accept([a], [list(range(60))])
    assert book.pages_in_use() == [0, 0] and whole(book)
    with pytest.raises(CacheMisuse):
        book.settle([a], [60])
    assert book.pages_in_use() == [0, 0] and whole(book)


class Meta:
    FEED = 8

    def upload(self, slots, *rest, **kw):
        return types.SimpleNamespace(T=len(slots), n=len(slots), max_count=1, fresh=False, ids_map=None, tree=None)


@pytest.mark.parametrize("step", ["token", "fed token", "tokens", "smaller tree"])
def test_pages_of_drafts_go_back_with_the_next_step(monkeypatch, step):
    """A sequence that takes another step than accepting holds the pages of that step alone; other sequences' drafts stay theirs."""
    from sleuth_b200.engine import stepper as module
    book = CacheBook([0, 100], 24, 2, stride=8)
    engine = bare_engine(book)
    s = engine.stepper
    model = types.SimpleNamespace(vocab=10, forward=lambda *a: None, logits=lambda *a: None)
    s.__dict__.update(model=model, device="cpu", max_len=512, max_step_tokens=64, meta=Meta(), use_graphs=False, ws=None, last_batch=None, _decode_logits=torch.zeros(8, 10),
                      _graphs={}, _seen_decode=set(), _raise_late_status=lambda: None, _look_at_status=lambda **kw: None, _draft_step=lambda b, parents: None,
                      _check_graph_key=lambda: None, max_graph_rows=64, max_draft_rows=512, portion=0)
    monkeypatch.setattr(module, "drafts_refusal", lambda model, cache: None)
    a, b = engine.open(2)
    book.grow([a, b], [60, 60])
    book.commit([a, b], [60, 60])
    for x in (a, b):
        drafted(engine, x, 200)
    assert book.pages_in_use() == [10, 10]
    if step == "token":
        engine.step([(a, [1], (0,))])
        assert int(book.lengths[a]) == 61
    elif step == "fed token":
        s.decode_fed([a], [0])
    elif step == "tokens":
        engine.step([(a, [1, 2, 3], ())])
        assert int(book.lengths[a]) == 63
    else:
        engine.step_tree([(a, [1, 2], [-1, 0])])
        assert s._drafted[a] == (60, 2)
    assert book.pages_in_use() == [6, 6] and whole(book)
    assert s._drafted[b] == (60, 200)
    engine.accept([b], [[0, 1]])
    assert book.pages_in_use() == [2, 2] and int(book.lengths[b]) == 62


def test_drafts_that_are_counted():
    """Proposals count, and those that were right; not the tokens that fill a step up to one width."""
    # one text repeats itself from the start, the other never, whose steps are filled up
    be = Drafting(lambda text, u: text[-1] % 4 + 1 if text[0] == 1 else text[-1] + 1, max_len=400, n_pages=64)
    circling, rising = generate_batches(be, [[1, 2, 3, 4] * 3, [50]], 24, SamplingConfig(temperature=0.0), stop_ids=(), max_batch=2, drafts=DraftPolicy(6))
    assert rising.stats["drafted"] == rising.stats["drafts_taken"] == 0 and rising.new_ids == list(range(51, 75))
    assert circling.stats["drafted"] == circling.stats["drafts_taken"] > 10
