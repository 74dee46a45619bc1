"""What a cache of bounded size asks of the host where its policy does not apply, and at the ends of its numbers (no GPU)."""

import numpy as np

from sleuth_b200.cache.book import CacheBook


def test_without_a_budget_tokens_and_rows_are_counted_once():
    """A step of many sequences sets each length once: with a count of its own beside it a commit of 64 sequences took the host 43 us, 13 without."""
    book = CacheBook([0, 100], n_pages=40, max_slots=4, stride=10, firsts=[0, 70])
    assert book.seen is book.lengths
    slots = book.open(3)
    for lens in ([5, 64, 1], [6, 65, 300], [7, 200, 301]):
        book.grow(slots, lens)
        book.commit(slots, lens)
        assert book.seen[slots].tolist() == book.lengths[slots].tolist() == lens
    book.close(slots)
    assert not book.lengths.any()
    bounded = CacheBook([0], n_pages=40, max_slots=4, stride=10, budget=70)
    s, = bounded.open(1)
    for rows, seen in ((60, 60), (100, 100), (71, 101), (72, 103)):
        bounded.grow([s], [rows])
        bounded.commit([s], [rows])
        assert (int(bounded.seen[s]), int(bounded.lengths[s])) == (seen, min(rows, 70))
    bounded.close([s])
    assert not np.any(bounded.seen) and not np.any(bounded.lengths)
