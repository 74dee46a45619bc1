"""The engine's steps of drafted tokens against the plain decoder, and generation with drafts against generation without."""

import numpy as np
import pytest
import torch

import tiny
import tiny_rabadra
from plain import qwen3_plain as plain

pytestmark = pytest.mark.gpu


# as the other engine tests, for the same weights: float32 sums in another order; bfloat16 activations rounded at every part
TOL = {"fp32": dict(rtol=1e-4, atol=2e-5), "bf16": dict(rtol=0.0, atol=1.7e-2)}


def _folder(tmp_path, name, **kw):
    import sleuth_b200 as sb
    sb.write_random_model(tmp_path, tiny.CONFIGS[name], seed=tiny.SEEDS[name], dtype=torch.float32, **kw)
    return tiny.CONFIGS[name]


def _way(parents, i):
    out = []
    while i >= 0:
        out.append(i)
        i = parents[i]
    return out[::-1]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("name", list("ABCDEFG"))
def test_steps_of_drafted_tokens(tmp_path, name, dtype):
    """Every node's logits are those of the text that ends with it; what is accepted goes on as if it had come token by token."""
    import sleuth_b200 as sb
    cfg = _folder(tmp_path, name)
    pc, pw = plain.read_model(tmp_path)
    if dtype == "bf16":
        pw = {k: v.to(torch.bfloat16).float() for k, v in pw.items()}
    rng = np.random.default_rng(3)
    longest = min(cfg["max_position_embeddings"], 256)
    engine = sb.load(tmp_path, dtype=dtype, max_seq_len=longest, device="cuda:0")
    texts = [rng.integers(0, cfg["vocab_size"], n).tolist() for n in (63, 5, 90)]
    slots = engine.open(3)
    engine.step([(s, t, ()) for s, t in zip(slots, texts)])
    got, want = [], []
    for turn in range(4):
        # (the same shape twice in a row and more: the third such step is a recorded one)
        trees = [[-1, 0, 0, 1, 2, 2, 3, 6], [-1, 0, 1, 2, 3, 4, 5, 6], [-1, 0, 0, 0, 2, 4, 5, 4]]
        tokens = [rng.integers(0, cfg["vocab_size"], len(t)).tolist() for t in trees]
        logits = engine.step_tree(list(zip(slots, tokens, trees))).cpu().double()
        at = 0
        for text, toks, tree in zip(texts, tokens, trees):
            for i in range(len(tree)):
                want.append(plain.logits(pc, pw, text + [toks[j] for j in _way(tree, i)])[-1].double())
            got.append(logits[at:at + len(tree)])
            at += len(tree)
        if turn == 2:      # nothing is accepted: the step might as well not have been
            continue
        ends = [7, 3, 6] if turn % 2 else [5, 7, 3]
        paths = [_way(tree, e) for tree, e in zip(trees, ends)]
        engine.accept(slots, paths)
        for text, toks, path in zip(texts, tokens, paths):
            text += [toks[j] for j in path]
    after = engine.step([(s, [1], (0,)) for s in slots]).cpu().double()
    got.append(after)
    want += [plain.logits(pc, pw, t + [1])[-1].double() for t in texts]
    got, want = torch.cat(got), torch.stack(want)
    torch.testing.assert_close(got, want, **TOL[dtype])
    engine.close(slots)


@pytest.mark.parametrize("name", ["A", "C", "D", "F"])
@pytest.mark.parametrize("temperature", [0.0, 0.9])
def test_generation_is_the_same_with_drafts(tmp_path, name, temperature):
    import sleuth_b200 as sb
    cfg = _folder(tmp_path, name, std=0.06)
    engine = sb.load(tmp_path, dtype="fp32", max_seq_len=128, device="cuda:0")
    rng = np.random.default_rng(4)
    phrase = rng.integers(0, cfg["vocab_size"], 9).tolist()
    prompts = [phrase * 3 + phrase[:4], rng.integers(0, cfg["vocab_size"], 20).tolist(), phrase[:2]]
    sampling = sb.SamplingConfig(temperature=temperature, top_k=5)
    plainly = engine.generate(prompts, 60, sampling, seed=2, stop_ids=())
    for policy in (sb.DraftPolicy(4), sb.DraftPolicy(9, 3, 2)):
        drafted = engine.generate(prompts, 60, sampling, seed=2, stop_ids=(), drafts=policy)
        # (float32 sums of several rows and of one agree to some 1e-6 of the logits, and no two logits of these texts lie so near)
        assert [r.new_ids for r in drafted] == [r.new_ids for r in plainly]
        assert [r.stop_reason for r in drafted] == [r.stop_reason for r in plainly]
    assert engine.cache.book.pages_in_use() == [0] * engine.cache.n_groups


def test_bfloat16_generation_with_drafts_runs(tmp_path):
    import sleuth_b200 as sb
    cfg = _folder(tmp_path, "G", std=0.06)
    engine = sb.load(tmp_path, dtype="bf16", max_seq_len=300, device="cuda:0")
    res = engine.generate([[3, 4, 5] * 10, [7] * 40], 200, sb.SamplingConfig(temperature=0.0), stop_ids=(), drafts=sb.DraftPolicy(6))
    assert [len(r.new_ids) for r in res] == [200, 200] and all(0 <= t < cfg["vocab_size"] for r in res for t in r.new_ids)
    assert sum(r.stats["drafts_taken"] for r in res) > 0


def test_refusals(tmp_path):
    import sleuth_b200 as sb
    from sleuth_b200.engine.engine import Engine
    _folder(tmp_path, "A")
    engine = sb.load(tmp_path, dtype="fp32", max_seq_len=64, device="cuda:0")
    slots = engine.open(2)
    engine.step([(s, [1, 2, 3], ()) for s in slots])
    for entry in ((slots[0], [1, 2], [-1]), (slots[0], [1, 2], [0, 0]), (slots[0], [1, 2], [-1, 1]), (slots[0], [1, 999], [-1, 0]), (slots[0], [], []),
                  (slots[0], [1, 2, 3], [-1, 0, -1])):
        with pytest.raises(ValueError):
            engine.step_tree([entry])
    with pytest.raises(RuntimeError, match="longest"):
        engine.step_tree([(slots[0], [1] * 62, [-1] + list(range(61)))])
    with pytest.raises(ValueError, match="accept"):
        engine.accept([slots[0]], [[0]])
    engine.step_tree([(slots[0], [1, 2, 3], [-1, 0, 0])])
    for path in ([], [1], [0, 3], [0, 2, 1]):
        with pytest.raises(ValueError, match="accept"):
            engine.accept([slots[0]], [path])
    engine.accept([slots[0]], [[0, 2]])
    with pytest.raises(ValueError, match="accept"):
        engine.accept([slots[0]], [[0]])
    assert engine.length(slots[0]) == 5 and engine.length(slots[1]) == 3
    engine.step_tree([(slots[0], [1, 2], [-1, 0])])
    engine.step([(slots[0], [5], (0,))])
    with pytest.raises(ValueError, match="accept"):      # another step since
        engine.accept([slots[0]], [[0]])
    kept = sb.load(tmp_path, dtype="fp32", max_seq_len=64, device="cuda:0", keep=sb.KeepPolicy(window=20))
    with pytest.raises(ValueError, match="drafts"):
        kept.generate([[1, 2]], 3, drafts=sb.DraftPolicy())
    other = Engine.from_config(tiny_rabadra.CONFIGS["A"], dtype="fp32", max_seq_len=64)
    with pytest.raises(ValueError, match="drafts"):
        other.step_tree([(other.open(1)[0], [1], [-1])])


@pytest.mark.parametrize("name,dtype", [("A", "fp32"), ("D", "fp32"), ("F", "fp32"), ("G", "bf16")])
@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_drafts_of_another_model(tmp_path, name, dtype, temperature):
    """The way of a program that drafts with a model of its own: step_tree, verify_drafts on its logits, accept, the chosen token as the next newest one. Every
    judgement is the definition's on these logits, and at temperature 0 the text is the one that single-token steps choose."""
    import sleuth_b200 as sb
    from plain import drafts_plain
    from sleuth_b200.kernels import ops
    cfg = _folder(tmp_path, name, std=0.06)
    vocab, dev = cfg["vocab_size"], "cuda:0"
    engine = sb.load(tmp_path, dtype=dtype, max_seq_len=128, device=dev)
    g, rng = torch.Generator().manual_seed(8), np.random.default_rng(8)
    prompts = [rng.integers(0, vocab, n).tolist() for n in (9, 30, 4)]
    slots = engine.open(3)
    newest = engine.step([(s, p, (len(p) - 1,)) for s, p in zip(slots, prompts)]).argmax(1).tolist()
    texts, taken = [[t] for t in newest], 0
    tree = [-1, 0, 0, 0, 1, 2, 4]
    n, c = len(slots), len(tree)
    T, i32 = n * c, lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    parents, starts, counts = i32(tree * n), i32([c * i for i in range(n)]), i32([c] * n)
    path, lengths, chosen = (torch.zeros(s, dtype=torch.int32, device=dev) for s in ((n, c), (n,), (n,)))
    scratch = torch.zeros(max(1, ops.verify_drafts_scratch_words(n, T, vocab, True)), dtype=torch.int32, device=dev)
    guess = engine.open(n)      # the drafting model: the same one, a token at a time, made to err now and then
    for s, p in zip(guess, prompts):
        engine.step([(s, p, ())])
    for _ in range(8):
        at = [engine.length(s) for s in guess]
        likely = engine.step([(s, t[-1:], (0,)) for s, t in zip(guess, texts)]).cpu()
        q = torch.softmax(2.0 * likely + torch.randn(likely.shape, generator=g), 1)
        probs = torch.zeros((T, vocab))
        tokens = torch.randint(0, vocab, (T,), generator=g, dtype=torch.int32)
        for i in range(n):
            tokens[c * i] = texts[i][-1]
            probs[c * i:c * i + c] = torch.softmax(torch.randn((c, vocab), generator=g), 1)
            probs[c * i] = q[i]
            tokens[c * i + 1:c * i + 4] = torch.multinomial(q[i], 3, replacement=True, generator=g).to(torch.int32)
        logits = engine.step_tree([(s, tokens[c * i:c * i + c].tolist(), tree) for i, s in enumerate(slots)])
        uniforms = torch.rand(T, generator=g)
        floors = torch.topk(logits, min(20, vocab), dim=1).values[:, -1].contiguous() if temperature else None
        ops.verify_drafts(logits, vocab, tokens.to(dev), parents, starts, counts, uniforms.to(dev), temperature, path, lengths, chosen, c, probs=probs.to(dev), floors=floors,
                          scratch=scratch)
        paths = [p[:k] for p, k in zip(path.tolist(), lengths.tolist())]
        for i in range(n):
            rows = slice(c * i, c * i + c)
            want = drafts_plain.verify(logits[rows].cpu(), tokens[rows], tree, uniforms[rows], temperature, vocab, probs[rows], None if floors is None else floors[rows].cpu())
            assert (paths[i], int(chosen[i])) == want
        engine.accept(slots, paths)
        more = [[int(tokens[c * i + k]) for k in p[1:]] + [int(chosen[i])] for i, p in enumerate(paths)]
        for s, text, m in zip(guess, texts, more):
            if len(m) > 1:
                engine.step([(s, m[:-1], ())])
            text += m
        taken += sum(len(m) - 1 for m in more)
        assert [engine.length(s) for s in guess] == [engine.length(s) for s in slots] == [a + len(m) for a, m in zip(at, more)]
    assert taken > 0
    engine.close(slots + guess)
    if temperature == 0.0 and dtype == "fp32":
        plainly = engine.generate(prompts, max(map(len, texts)), sb.SamplingConfig(temperature=0.0), stop_ids=())
        # (float32 sums of several rows and of one agree to some 1e-6 of the logits, and no two logits of these texts lie so near)
        assert [r.new_ids[:len(t)] for r, t in zip(plainly, texts)] == texts


@pytest.mark.parametrize("name", ["A", "E", "G"])
@pytest.mark.parametrize("policy", [(6, 1, 3), (9, 3, 1)], ids=str)
def test_bfloat16_choices_with_drafts(tmp_path, name, policy):
    """In bfloat16 a step of several tokens rounds otherwise than one of a single token: a choice is the plain decoder's wherever its two largest logits lie further
    apart than both sides' rounding."""
    import sleuth_b200 as sb
    cfg = _folder(tmp_path, name)
    pc, pw = plain.read_model(tmp_path)
    pw = {k: v.to(torch.bfloat16).float() for k, v in pw.items()}
    longest = min(cfg["max_position_embeddings"], 200)
    engine = sb.load(tmp_path, dtype="bf16", max_seq_len=longest, device="cuda:0")
    rng = np.random.default_rng(5)
    phrase = rng.integers(0, cfg["vocab_size"], 7).tolist()
    prompts = [phrase * 4, phrase[:3] * 9 + phrase, rng.integers(0, cfg["vocab_size"], 12).tolist() * 2]
    res = engine.generate(prompts, 40, sb.SamplingConfig(temperature=0.0), stop_ids=(), drafts=sb.DraftPolicy(*policy))
    assert sum(r.stats["drafted"] for r in res) > 0
    for r in res:
        rows = plain.logits(pc, pw, r.prompt_ids + r.new_ids)[len(r.prompt_ids) - 1:-1].double()
        short = rows.max(1).values - rows.gather(1, torch.tensor(r.new_ids)[:, None])[:, 0]
        assert bool((short <= 2 * TOL["bf16"]["atol"]).all()), float(short.max())
