"""What a cache of bounded size asks of the host where its policy does not apply, and at the ends of its numbers (no GPU)."""

import numpy as np
import pytest
import torch

import tiny
from sleuth_b200.cache.book import CacheBook
from sleuth_b200.cache.keep import KeepPolicy
from sleuth_b200.config.registry import parse_config
from sleuth_b200.engine.engine import _cache_for
from sleuth_b200.engine.model import Model
from sleuth_b200.parts.base import BuildContext


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


def test_a_sequence_holds_no_more_rows_than_its_text_has_tokens():
    """``portion`` without a limit, a budget above every text: what the cache reserves goes by the longest text then."""
    most = 2 ** 31 - 1
    assert KeepPolicy(budget=2048).rows_for(32768) == 2560
    assert KeepPolicy(budget=2048).rows_for(1000) == 1000
    assert KeepPolicy(budget=100, portion=most).rows_for(4096) == 4096
    assert KeepPolicy(budget=most).rows_for(4096) == 4096
    arch, cfg, _ = parse_config(tiny.CONFIGS["A"])
    spec = arch.model_spec(cfg)
    for policy, longest, rows in ((KeepPolicy(budget=most, portion=most), 320, 320), (KeepPolicy(budget=70, portion=60), 4096, 192), (KeepPolicy(budget=70, portion=60), 100, 128)):
        model = Model(spec, BuildContext(device="cpu", dtype=torch.float32, max_positions=-(-longest // 64) * 64, keep=policy))
        shapes = {name: getattr(r, "shape", None) for name, r in model.cache_requests[0].parts}
        cache = _cache_for(model, policy, None, longest, torch.float32, "cpu", 2)
        assert shapes["gathered"] == shapes["positions"] == (cfg.kv_heads, rows) and cache.stride * 64 == rows


@pytest.mark.parametrize("name", ["budget", "window", "first", "portion"])
def test_numbers_that_no_row_can_have_are_refused_at_once(name):
    kw = dict(budget=50) if name in ("first", "portion") else {}
    with pytest.raises(ValueError):
        KeepPolicy(**{**kw, name: 2 ** 31})
    with pytest.raises(ValueError):
        KeepPolicy(budget=50, recent=2 ** 31)


def test_the_command_line_reserves_state_for_its_prompts_alone(monkeypatch):
    from sleuth_b200 import cli
    from sleuth_b200.engine import engine

    class Loaded(Exception):
        pass

    def load(path, **kw):
        raise Loaded(kw)

    monkeypatch.setattr(engine, "load", load)

    def asked(*options):
        with pytest.raises(Loaded) as e:
            cli.main(["generate", "m", "--prompt-ids", "1 2; 3 4 5", *options])
        return e.value.args[0]

    kw = asked("--keep-budget", "2048")
    assert kw["max_sequences"] == 2 and kw["max_tokens"] == 2 * 2560 and kw["keep"].budget == 2048
    assert asked("--keep-window", "100")["max_sequences"] == 2
    assert asked()["max_sequences"] is None and asked()["keep"] is None


def test_the_command_line_does_not_ignore_half_a_policy():
    from sleuth_b200 import cli
    with pytest.raises(ValueError):
        cli.main(["generate", "m", "--prompt-ids", "1 2", "--keep-recent", "100"])


@pytest.mark.parametrize("name", ["q", "k_pool", "block_table", "weights"])
@pytest.mark.parametrize("rank", [0, 1])
def test_operators_name_arguments_of_another_rank(name, rank):
    """Told before anything is launched or asked of a device."""
    from sleuth_b200.kernels import ops
    odd = torch.zeros(()) if rank == 0 else torch.zeros(8)
    i32 = torch.zeros(1, dtype=torch.int32)
    pool, table, w = torch.zeros((2, 2, 64, 16)), torch.zeros((1, 2), dtype=torch.int32), torch.zeros((1, 2, 128))
    attend = {**dict(q=torch.zeros((1, 4, 16)), k_pool=pool, block_table=table, weights=w), name: odd}
    with pytest.raises(ValueError, match="attention_kept"):
        ops.attention_kept(v_pool=pool, out=torch.zeros((1, 64)), seq_start=i32, past=i32, counts=i32, max_count=1, heads=4, kv_heads=2, head_dim=16, window=0,
                           first=0, scale=1.0, **attend)
    if name != "q":
        evict = {**dict(k_pool=pool, block_table=table, weights=w), name: odd}
        with pytest.raises(ValueError, match="cache_evict"):
            ops.cache_evict(positions=w.int(), v_pool=pool, past=i32, lengths=i32, seen=i32, budget=3, first=0, recent=0, **evict)
