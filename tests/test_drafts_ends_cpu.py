"""Steps of drafted tokens that nobody accepts: slots that were closed, pages that were taken, drafts that were counted. No GPU."""

import types

import pytest

from sleuth_b200.cache.book import CacheBook, CacheMisuse
from sleuth_b200.engine.engine import Engine
from sleuth_b200.engine.stepper import Stepper


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
