"""The generation loop with drafted tokens, with a scripted backend instead of a GPU: the same tokens, reasons and ends as without drafts."""

import random

import pytest

from sleuth_b200.cache.book import CacheBook, CacheMisuse
from sleuth_b200.engine.generate import generate_batches
from sleuth_b200.sampling import DraftPolicy, NgramDrafter, SamplingConfig

from test_generate_loop import ScriptedBackend


class Drafting(ScriptedBackend):
    """Its "logits" are texts: the next token of a text is script(text)."""
    pipelined = False

    def __init__(self, script, **kw):
        super().__init__(lambda prompt, k: None, **kw)
        self.next = script
        self.trees = 0

    def _append(self, slots, lists):
        super()._append(slots, lists)
        return [tuple(self.seq[s]) for s in slots]

    def step_tree(self, entries):
        out, self.pending = [], {}
        slots = [s for s, _, _ in entries]
        new = [int(self.book.lengths[s]) + len(t) for s, t, _ in entries]
        assert all(n <= self.max_len for n in new), "the loop stepped past the context"
        self.book.grow(slots, new)
        for s, tokens, parents in entries:
            ways = []
            for t, p in zip(tokens, parents):
                ways.append((ways[p] if p >= 0 else ()) + (t,))
            out += [tuple(self.seq[s]) + w for w in ways]
            self.pending[s] = tokens
        self.trees += 1
        return out

    def accept(self, slots, paths):
        self.book.settle(slots, [int(self.book.lengths[s]) + len(p) for s, p in zip(slots, paths)])
        for s, path in zip(slots, paths):
            assert path[0] == 0 and all(a < b for a, b in zip(path, path[1:]))
            self.seq[s].extend(self.pending[s][i] for i in path)

    def choose(self, logits, cfg, uniforms, vocab_limit, recent, banned):
        us = [0.0] * len(logits) if uniforms is None else uniforms
        return [self.next(text, u) for text, u in zip(logits, us)]


def repeating(text, u):
    """A text that goes in circles with a random step aside now and then."""
    return (text[-1] * 5 + len(text) // 17 + (1 if u > 0.8 else 0)) % 23


def circling(text, u):
    """A text that comes round every six tokens, with a random step aside now and then."""
    return (text[-1] * 5 + (1 if u > 0.95 else 0)) % 7 if len(text) % 120 else 22


@pytest.mark.parametrize("script", [repeating, circling])
@pytest.mark.parametrize("policy", [DraftPolicy(1, 1, 1), DraftPolicy(4), DraftPolicy(8, 3, 2), DraftPolicy(30, 5, 4)], ids=str)
@pytest.mark.parametrize("temperature", [0.0, 1.0])
@pytest.mark.parametrize("kw", [dict(max_len=200, n_pages=64), dict(max_len=64, n_pages=64), dict(max_len=128, n_pages=4), dict(max_len=300, n_pages=3, max_slots=3)], ids=str)
def test_drafts_change_nothing(policy, temperature, kw, script):
    rng = random.Random(3)
    prompts = [[rng.randrange(23) for _ in range(n)] for n in (1, 30, 61, 7, 64)]
    for new in (1, 2, 9, 150):
        runs = []
        for drafts in (None, policy):
            be, seen = Drafting(script, **kw), []
            got = generate_batches(be, prompts, new, SamplingConfig(temperature=temperature), stop_ids={22}, seed=5, max_batch=3, drafts=drafts,
                                   on_token=lambda r, t: seen.append((r, t)))
            assert be.book.free_slots == be.book.max_slots and be.book.pages_in_use() == [0]
            runs.append((got, sorted(seen, key=lambda x: x[0]), be))
        for a, b in zip(runs[0][0], runs[1][0]):
            assert (a.new_ids, a.stop_reason, a.prompt_ids) == (b.new_ids, b.stop_reason, b.prompt_ids)
        assert runs[0][1] == runs[1][1]
        if new == 150 and policy.tokens > 1 and kw["max_len"] == 200 and script is circling:
            assert runs[1][2].trees > 0 and sum(r.stats["drafts_taken"] for r in runs[1][0]) > 50


@pytest.mark.parametrize("most", [3, 4, 7, 20])
def test_a_step_brings_no_more_tokens_than_the_backend_takes(most):
    prompts, runs = [[1, 2, 3] * 5, [4] * 9, [5, 6] * 6], []
    for drafts in (None, DraftPolicy(8, 2)):
        be = Drafting(circling, max_len=200, n_pages=64)
        be.max_step_tokens, step, widest = most, be.step_tree, []
        be.step_tree = lambda entries: (widest.append(sum(len(t) for _, t, _ in entries)), step(entries))[1]
        runs.append([r.new_ids for r in generate_batches(be, prompts, 90, SamplingConfig(temperature=0.0), stop_ids={22}, seed=5, max_batch=3, drafts=drafts)])
    assert runs[0] == runs[1] and max(widest, default=0) <= most and (most < 6 or widest)


def test_drafts_and_penalties_do_not_go_together():
    with pytest.raises(ValueError, match="drafts"):
        generate_batches(Drafting(repeating), [[1]], 3, SamplingConfig(repetition_penalty=1.2), drafts=DraftPolicy())


def test_policies_that_make_no_sense_are_refused():
    for kw in (dict(tokens=0), dict(tokens=256), dict(branches=0), dict(ngram=0), dict(tokens=True), dict(tokens=2.0)):
        with pytest.raises(ValueError, match="drafts"):
            DraftPolicy(**kw)


def test_lookups():
    d = NgramDrafter(DraftPolicy(5, 2, 3), [1, 2, 3, 4, 9, 2, 3, 5, 6, 7, 2, 3])
    # "2 3" was followed by 5 6 7 2 3, and before that by 4 9 2 3 5: the latest first, then another branch, as far as there is room
    assert d.propose(10) == ([5, 6, 7, 2, 3], [0, 1, 2, 3, 4])
    assert d.propose(3) == ([5, 6, 7], [0, 1, 2])
    assert NgramDrafter(DraftPolicy(6, 2, 3), [1, 2, 3, 4, 9, 2, 3, 5, 2, 3]).propose(9) == ([5, 2, 3, 4, 9, 2], [0, 1, 2, 0, 4, 5])
    assert d.propose(0) == ([], []) and NgramDrafter(DraftPolicy(), [1, 2, 3]).propose(5) == ([], [])
    assert NgramDrafter(DraftPolicy(4, 1, 3), [7, 7]).propose(9) == ([7], [0])
    rng = random.Random(1)
    for _ in range(300):
        text = [rng.randrange(4) for _ in range(rng.randrange(1, 60))]
        policy = DraftPolicy(rng.randrange(1, 20), rng.randrange(1, 5), rng.randrange(1, 5))
        tokens, parents = NgramDrafter(policy, text).propose(rng.randrange(0, 25))
        assert len(tokens) == len(parents) <= policy.tokens and all(0 <= p <= i for i, p in enumerate(parents))
        siblings = list(zip(parents, tokens))
        assert len(set(siblings)) == len(siblings)


def test_pages_behind_what_is_kept_go_back():
    book = CacheBook([0, 40], 8, 2, stride=4)
    a, b = book.open(2)
    book.grow([a, b], [60, 10])
    book.commit([a, b], [60, 10])
    book.grow([a, b], [150, 70])
    assert book.pages_in_use() == [5, 5]
    book.settle([a, b], [65, 11])
    assert book.pages_in_use() == [3, 3] and book.lengths[a] == 65 and book.lengths[b] == 11
    book.grow([a], [200])
    book.settle([a], [140])
    assert book.pages_in_use()[0] == 4 and book.pages_in_use()[1] == 3      # (the window of 40 has moved past the first page)
    book.close([a, b])
    assert book.pages_in_use() == [0, 0]
    bounded = CacheBook([0], 8, 1, stride=4, budget=32)
    with pytest.raises(CacheMisuse):
        bounded.settle(bounded.open(1), [1])
