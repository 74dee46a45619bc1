"""The engine over a cache of bounded size against the plain decoder in 64 bits under the same policy."""

import numpy as np
import pytest
import torch

import tiny
from plain import keep_plain, qwen3_plain as plain

pytestmark = pytest.mark.gpu

WINDOW = dict(window=50, first=5)
CASES = [("A", dict(budget=24, first=2, recent=8, portion=16)), ("B", dict(budget=40, first=0, portion=30)), ("D", dict(budget=70, first=4, recent=20, portion=60)),
         ("G", dict(budget=66, first=3, recent=0, portion=200)), ("A", dict(window=9, first=1)), ("B", WINDOW), ("D", dict(window=100, first=70)), ("G", WINDOW)]


def _portions(policy, n):
    if not policy.budget:
        return [n]
    return [min(policy.portion, n - i) for i in range(0, n, policy.portion)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("name,kw", CASES, ids=[f"{n}-{'budget' if 'budget' in k else 'window'}" for n, k in CASES])
def test_prompts_and_tokens(tmp_path, name, kw, dtype):
    import sleuth_b200 as sb
    cfg = tiny.CONFIGS[name]
    # larger weights than the other tests': scores that differ, so that some rows are looked at much more than others
    sb.write_random_model(tmp_path, cfg, seed=tiny.SEEDS[name], dtype=torch.float32, std=0.06)
    policy = sb.KeepPolicy(**kw)
    pc, pw = plain.read_model(tmp_path)
    if dtype == "bf16":
        pw = {k: v.to(torch.bfloat16).float() for k, v in pw.items()}
    rng = np.random.default_rng(5)
    longest = min(cfg["max_position_embeddings"], 300)
    lengths = [longest - 12, 5, 33]
    prompts = [rng.integers(0, cfg["vocab_size"], n).tolist() for n in lengths]
    later = rng.integers(0, cfg["vocab_size"], (8, 3)).tolist()
    texts = [keep_plain.Text(pc, pw, policy) for _ in prompts]
    engine = sb.load(tmp_path, dtype=dtype, max_seq_len=longest, device="cuda:0", keep=policy)
    slots = engine.open(3)
    got = [engine.step([(s, p, (len(p) - 1,)) for s, p in zip(slots, prompts)]).cpu().double()]
    want = []
    for t, p in zip(texts, prompts):
        at = 0
        for n in _portions(policy, len(p)):
            row = t.append(p[at:at + n])[-1]
            at += n
        want.append(row)
    want = [torch.stack(want)]
    for step in later:
        got.append(engine.step([(s, (t,), (0,)) for s, t in zip(slots, step)]).cpu().double().clone())
        want.append(torch.stack([t.append([tok])[-1] for t, tok in zip(texts, step)]))
    # a short turn at the end: several tokens at once behind what is held
    turn = rng.integers(0, cfg["vocab_size"], 3).tolist()
    got.append(engine.step([(slots[1], turn, (2,))]).cpu().double())
    want.append(texts[1].append(turn)[-1:])
    scale = float(torch.cat(want).abs().max())
    if policy.budget and dtype == "fp32":
        # the same rows stay, in the same places, unless an eviction was as close as the rounding of the sums
        assert min(t.gap for t in texts) > 1e-5, "choose another seed: an eviction is too close a call for 32 bits"
        for layer in range(cfg["num_hidden_layers"]):
            view = engine.cache.view(layer, writes=True)
            for s, t in zip(slots, texts):
                for kh in range(cfg["num_key_value_heads"]):
                    r = t.rows[layer][kh]
                    assert engine.cache.book.lengths[s] == len(r["at"]) and engine.length(s) == t.seen
                    assert view["positions"].state[s, kh, :len(r["at"])].tolist() == r["at"]
                    w = view["gathered"].state[s, kh, :len(r["at"])].cpu().double()
                    assert torch.allclose(w, torch.tensor(r["w"], dtype=torch.float64), rtol=1e-4, atol=1e-5)
    # float32: sums of a few hundred products through 2 or 3 layers, 1e-5 of the logits' size each at most. bfloat16: every product, key and value
    # is rounded to 2^-9, some forty roundings on the way that partly cancel; under a budget a close call may also keep another row
    rel = 2e-4 if dtype == "fp32" else 0.06
    for g, w in zip(got, want):
        assert float((g - w).abs().max()) <= rel * scale
    engine.stepper.check_status()
    engine.close(slots)
    assert engine.cache.book.pages_in_use() == [0]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_a_budget_above_the_text_changes_nothing_but_the_order_of_sums(tmp_path, dtype):
    import sleuth_b200 as sb
    cfg = tiny.CONFIGS["D"]
    sb.write_random_model(tmp_path, cfg, seed=9, dtype=torch.float32)
    prompts = [np.random.default_rng(1).integers(0, cfg["vocab_size"], n).tolist() for n in (70, 9)]
    rows = []
    for keep in (None, sb.KeepPolicy(budget=400, portion=64), sb.KeepPolicy(window=500, first=4)):
        engine = sb.load(tmp_path, dtype=dtype, max_seq_len=300, device="cuda:0", keep=keep)
        slots = engine.open(2)
        out = [engine.step([(s, p, (len(p) - 1,)) for s, p in zip(slots, prompts)]).cpu()]
        for i in range(4):
            out.append(engine.step([(s, (i + 3,), (0,)) for s in slots]).cpu().clone())
        rows.append(torch.cat(out))
    for r in rows[1:]:
        assert float((r - rows[0]).abs().max()) <= (1e-5 if dtype == "fp32" else 0.03) * float(rows[0].abs().max())


def test_generates_far_beyond_what_the_cache_holds(tmp_path):
    import sleuth_b200 as sb
    cfg = tiny.CONFIGS["D"]
    sb.write_random_model(tmp_path, cfg, seed=9, dtype=torch.float32)
    prompts = [np.random.default_rng(i).integers(0, cfg["vocab_size"], n).tolist() for i, n in enumerate((300, 40, 3))]
    for keep, tokens in ((sb.KeepPolicy(budget=64, portion=64), 3 * 128), (sb.KeepPolicy(window=64, first=4), 1024)):
        engine = sb.load(tmp_path, dtype="bf16", max_seq_len=600, max_tokens=tokens, device="cuda:0", keep=keep)
        out = engine.generate(prompts, max_new_tokens=200, sampling=sb.SamplingConfig(temperature=0.0), stop_ids=())
        assert [len(r.new_ids) for r in out] == [200, 200, 200]
        again = engine.generate(prompts, max_new_tokens=200, sampling=sb.SamplingConfig(temperature=0.0), stop_ids=(), cuda_graph=False)
        assert [r.new_ids for r in out] == [r.new_ids for r in again]
    with pytest.raises(ValueError):
        sb.load(tmp_path, keep=sb.KeepPolicy(budget=3, recent=9))
    sb.write_random_model(tmp_path / "w", tiny.CONFIGS["E"], seed=9, dtype=torch.float32)
    with pytest.raises(ValueError):
        sb.load(tmp_path / "w", keep=sb.KeepPolicy(window=9))
