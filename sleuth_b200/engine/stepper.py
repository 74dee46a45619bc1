"""The step function: run the tokens a batch brings, from the cache, and return the wanted logits.

A step takes sequences that start together (their prompts, of unequal lengths) or go on together
(one token each); in fact each sequence may bring any number of tokens, and they are appended after
what its slot already holds. Only the given tokens are computed. Every sequence's keys and values go
to its own pages and every query reads its own sequence's pages, so no padding exists and nothing a
sequence computes depends on the others in the batch.

The reference's counterpart is ``Transformer.forward(idx, cache)`` with one shared position for a
rectangular batch and logits for every position (sleuth/forge/model/transformer.py:257-313,
sleuth/forge/infer/kv_cache.py:34,62-64); ragged batches, per-sequence positions and logits at chosen
rows only are this library's own.

Long steps are cut into chunks of at most ``max_step_tokens`` tokens; a chunk runs through all
layers before the next begins, so later chunks of a sequence find the earlier ones in the cache.
A step in which every sequence brings one token is replayed as a CUDA graph from its second
occurrence at a batch size on (the reference captures one decode step per length bucket,
sleuth/forge/infer/cuda_graph.py:96-129; here lengths live in device tables, so one graph per batch
size serves every length).
"""

from __future__ import annotations

from dataclasses import dataclass

import os

import numpy as np
import torch

from ..cache.book import CacheFull
from ..kernels import ops
from ..parts.attention import GQAAttention
from ..parts.base import Workspace
from ..parts.ends import TokenEmbedding
from .batch import MetaStager


@dataclass
class StepEntry:
    slot: int
    tokens: object              # sequence of token ids
    want: object = ()           # positions among ``tokens`` whose logits are wanted


@dataclass
class TreeEntry:
    """A sequence's share of a step of drafted tokens: ``tokens[0]`` is its newest certain token, ``tokens[i]`` a draft behind ``tokens[parents[i]]``
    (``parents[i]`` < i; ``parents[0]`` is -1)."""
    slot: int
    tokens: object
    parents: object


@dataclass
class DraftStep:
    """What the attention parts need of such a step."""
    positions: torch.Tensor         # [tokens] int32, by which rows are rotated
    seen: list                      # per cache group [tokens, words] int32: the rows of the step that a row sees under the group's window


def drafts_refusal(model, cache) -> str | None:
    """Why steps of drafted tokens are not built for a model, or None."""
    if cache.book.budget:
        return "a cache with a budget gives no rows back"
    if type(model.embedding) is not TokenEmbedding or model.embedding.turns is not None:
        return "the embedding is more than a table of tokens"
    mixers = [layer.children.get("mixer") if hasattr(layer, "children") else None for layer in model.layers]
    if not all(isinstance(m, GQAAttention) and m.takes_drafts for m in mixers):
        return "every mixer has to be grouped-query attention over a cache entry of its own, without a policy, chunks, sinks, a gate or values of another width"
    schedule = model.spec.schedule
    if len({e.cache for e in schedule}) != len(schedule) or any(e.borrow >= 0 for e in schedule):
        return "layer applications share a cache entry"
    return None


class Stepper:
    STATUS_EVERY = 16

    def __init__(self, model, cache, device, max_len: int | None = None, max_step_tokens: int = 8192,
                 use_graphs: bool = True, max_graph_batch: int = 256, portion: int = 0):
        """portion: the most tokens one sequence may bring in a chunk (0: no limit), which a cache with a budget needs: its
        rows are bounded by the budget and one portion, whatever the length of the texts."""
        self.model, self.cache = model, cache
        self.portion = int(portion)
        budget = cache.book.budget
        self.max_len = cache.book.max_len if max_len is None else int(max_len) if budget else min(int(max_len), cache.book.max_len)
        self.device = torch.device(device)
        self.max_step_tokens = max_step_tokens
        self.use_graphs = use_graphs
        self.max_graph_batch = max_graph_batch
        self.ws = Workspace(self.device)
        self.meta = MetaStager(self.device, cache.n_groups, cache.stride, rows_apart=budget > 0)
        self._graphs: dict = {}
        self._seen_decode: set = set()
        self._seen_chunk: set = set()
        self._chunk_logits: torch.Tensor | None = None
        self.max_graph_rows = 64        # steps of many tokens are recorded only if they want at most this many rows of logits
        self.max_draft_rows = 512       # the same for steps of drafted tokens, which want every row's
        self.max_chunk_graphs = 16      # recordings of such steps kept at a time
        self._decode_logits: torch.Tensor | None = None
        self._graph_key = None
        self.check_kernels = os.environ.get("SLEUTH_B200_CHECK", "0") == "1"   # read the kernels' status word after each step
        self._status_host: torch.Tensor | None = None     # pinned copy of the kernels' status word, read one step late
        self._status_event = None
        self._steps_unseen = 0              # single-token steps since the word was last copied
        self._graph_own: dict = {}          # own kernel launches captured in each graph
        self.graph_kernel_launches = 0      # own kernel launches replayed through graphs so far
        self._drafted: dict[int, tuple[int, int]] = {}      # slot -> its rows before the last step of drafted tokens, and the rows of that step
        self._draft_parents: torch.Tensor | None = None     # what a recorded step of drafted tokens reads, at fixed places
        self._draft_tables: dict = {}
        ops.lib()   # build or load the kernels now; fail here, loudly, if that is impossible

    # ------------------------------------------------------------------ public ----
    def step(self, entries: list[StepEntry], floats: np.ndarray | None = None) -> torch.Tensor:
        """Run one step. Returns float32 logits ``[sum(len(e.want)), vocab]`` in the order of the
        entries and of their ``want``. After a step of single tokens the result may be a view of a
        buffer that the next step overwrites."""
        if not entries:
            return torch.empty((0, self.model.vocab), dtype=torch.float32, device=self.device)
        self._raise_late_status()
        toks = [np.asarray(e.tokens, dtype=np.int64).reshape(-1) for e in entries]
        book = self.cache.book
        for e, t in zip(entries, toks):
            if t.size == 0:
                raise ValueError(f"slot {e.slot}: a step must bring at least one token for every sequence")
            if t.min() < 0 or t.max() >= self.model.vocab:
                raise ValueError(f"slot {e.slot}: token ids must lie in [0, {self.model.vocab})")
            for w in e.want:
                if not 0 <= int(w) < t.size:
                    raise ValueError(f"slot {e.slot}: wanted position {w} is outside its {t.size} tokens")
        slots = [int(e.slot) for e in entries]
        if len(set(slots)) != len(slots):
            raise ValueError("a step names a slot twice")
        finals = [int(book.seen[s]) + int(t.size) for s, t in zip(slots, toks)]
        for s, n in zip(slots, finals):
            if n > self.max_len:
                raise CacheFull(f"slot {s} would hold {n} tokens; the longest sequence allowed is {self.max_len}")

        if all(t.size == 1 for t in toks):
            return self._decode(entries, slots, toks, floats)

        chunks = self._cut(toks)
        # All or nothing: a step that the cache cannot hold to its end is refused before its first chunk runs, so a
        # sequence is never left half-appended.
        lens = {s: int(book.lengths[s]) for s in slots}
        plan = []
        for chunk in chunks:
            c_slots = [slots[i] for i, _, _ in chunk]
            for (i, _, take), s in zip(chunk, c_slots):
                lens[s] += take
            plan.append((c_slots, [lens[s] for s in c_slots]))
            if book.budget:
                for s in c_slots:
                    lens[s] = min(lens[s], book.budget)
        for g, need in zip(book.groups, book.peak_pages_needed(plan)):
            if need > g.pool.free:
                raise CacheFull(f"the step needs {need} more pages of 64 tokens and {g.pool.free} of {g.pool.n_pages} "
                                f"are free; nothing of it was run")

        n_want = sum(len(e.want) for e in entries)
        out = torch.empty((n_want, self.model.vocab), dtype=torch.float32, device=self.device)
        out_base, acc = [], 0
        for e in entries:
            out_base.append(acc)
            acc += len(e.want)
        for chunk in chunks:
            self._run_chunk(entries, slots, toks, chunk, out, out_base)
        self._look_at_status()
        return out

    # ------------------------------------------------------------------ drafted tokens ----
    def step_tree(self, entries: list[TreeEntry]) -> torch.Tensor:
        """Run the newest token of each sequence and the drafts behind it, all at once: float32 logits of every node, in the order of the entries and
        of their tokens. Nothing of it is kept until ``accept`` says which nodes are; a sequence that takes another step before is as it was,
        its pages too (until then, or until it is closed, it holds those of the drafts)."""
        why = drafts_refusal(self.model, self.cache)
        if why is not None:
            raise ValueError(f"drafts: not built for this model: {why}")
        if not entries:
            return torch.empty((0, self.model.vocab), dtype=torch.float32, device=self.device)
        self._raise_late_status()
        book = self.cache.book
        toks = [np.asarray(e.tokens, dtype=np.int64).reshape(-1) for e in entries]
        trees = [np.asarray(e.parents, dtype=np.int64).reshape(-1) for e in entries]
        slots = [int(e.slot) for e in entries]
        if len(set(slots)) != len(slots):
            raise ValueError("a step names a slot twice")
        for s, t, p in zip(slots, toks, trees):
            if not 1 <= t.size <= ops.MOST_NODES or p.size != t.size:
                raise ValueError(f"slot {s}: a step of drafted tokens brings 1 to {ops.MOST_NODES} tokens and a parent for each")
            if t.min() < 0 or t.max() >= self.model.vocab:
                raise ValueError(f"slot {s}: token ids must lie in [0, {self.model.vocab})")
            if p[0] != -1 or (t.size > 1 and (p[1:].min() < 0 or (p[1:] >= np.arange(1, t.size)).any())):
                raise ValueError(f"slot {s}: a draft continues an earlier token of the step, and the first token none (-1)")
        past = [int(book.lengths[s]) for s in slots]
        counts = [int(t.size) for t in toks]
        new_lens = [p + c for p, c in zip(past, counts)]
        for s, n in zip(slots, new_lens):
            if n > self.max_len:
                raise CacheFull(f"slot {s} would hold {n} tokens; the longest sequence allowed is {self.max_len}")
        T = sum(counts)
        if T > self.max_step_tokens:
            raise ValueError(f"a step of drafted tokens brings at most {self.max_step_tokens} tokens, got {T}")
        book.grow(slots, new_lens)
        self._drop_drafts(slots, new_lens)
        b = self.meta.upload(slots, past, counts, np.concatenate(toks).astype(np.int32), np.arange(T, dtype=np.int32), book.tables_for(slots))
        b.tree = self._draft_step(b, np.concatenate(trees).astype(np.int32))
        out = torch.empty((T, self.model.vocab), dtype=torch.float32, device=self.device)
        if not self._chunk_by_graph(b, T, out, np.arange(T)):
            self.model.forward(b, self.cache, self.ws, out)
        for s, p, c in zip(slots, past, counts):
            self._drafted[s] = (p, c)
        self._look_at_status()
        return out

    def _draft_step(self, b, parents: np.ndarray) -> DraftStep:
        """The step's parents on the device, and the tables that the attention reads, one launch a window."""
        T, words = b.T, -(-b.max_count // 32)
        if self._draft_parents is None or self._draft_parents.numel() < T:
            self._draft_parents = torch.zeros(max(2 * T, 1024), dtype=torch.int32, device=self.device)
            self._draft_tables.clear()
            self._graphs.clear()
        at = self._draft_parents[:T]
        at.copy_(torch.from_numpy(parents))
        if words not in self._draft_tables:
            cap = self._draft_parents.numel()
            windows = sorted({r.window for r in self.cache.group_requests})
            self._draft_tables[words] = (torch.zeros(cap, dtype=torch.int32, device=self.device),
                                         {w: torch.zeros((cap, words), dtype=torch.int32, device=self.device) for w in windows})
        positions, seen = self._draft_tables[words]
        for window, table in seen.items():
            ops.draft_tree(at, b.seq_start, b.past, b.counts, table, positions, b.max_count, window)
        return DraftStep(positions, [seen[r.window] for r in self.cache.group_requests])

    def forget(self, slots) -> None:
        """Slots that were closed, or stand for new sequences: what an earlier one drafted is not theirs to accept."""
        for s in slots:
            self._drafted.pop(int(s), None)

    def _drop_drafts(self, slots, lengths) -> None:
        """``slots`` take another step, after which they hold ``lengths`` rows: what they drafted goes, and the pages that only drafts had."""
        if self._drafted:
            for s, n in zip(slots, lengths):
                if self._drafted.pop(s, None) is not None:
                    self.cache.book.trim([s], [n])

    def accept(self, slots, paths) -> None:
        """Of the last ``step_tree`` of each of ``slots`` the nodes of its path stay (numbers of its tokens, rising, from 0 on); their rows move together in every
        layer and the others' go."""
        book = self.cache.book
        slots = [int(s) for s in slots]
        paths = [[int(i) for i in p] for p in paths]
        if len(set(slots)) != len(slots) or len(paths) != len(slots):
            raise ValueError("accept: one path for each slot, every slot once")
        for s, p in zip(slots, paths):
            past, count = self._drafted.get(s, (-1, 0))
            if past < 0 or past != int(book.lengths[s]):
                raise ValueError(f"accept: slot {s} has taken no step of drafted tokens, or another one since")
            if not p or p[0] != 0 or any(a >= b for a, b in zip(p, p[1:])) or p[-1] >= count:
                raise ValueError(f"accept: slot {s}: a path rises from 0 and stays below the step's {count} tokens")
        moving = [i for i, p in enumerate(paths) if p != list(range(len(p)))]
        if moving:
            width = max(len(paths[i]) for i in moving)
            host = np.full((len(moving), width + 2), -1, dtype=np.int32)
            for row, i in zip(host, moving):
                row[:len(paths[i])] = paths[i]
                row[width:] = book.lengths[slots[i]], len(paths[i])
            both = torch.from_numpy(host).to(self.device)
            path, past, lengths = (both[:, a:z].contiguous() for a, z in ((0, width), (width, width + 1), (width + 1, width + 2)))
            for pool, rows in zip(self.cache.pools, book.tables_for([slots[i] for i in moving])):
                ops.cache_compact(pool, torch.from_numpy(np.ascontiguousarray(rows)).to(self.device), past, path, lengths)
        for s in slots:
            del self._drafted[s]
        book.settle(slots, [int(book.lengths[s]) + len(p) for s, p in zip(slots, paths)])

    def _cut(self, toks) -> list:
        """The chunks of a step: lists of (entry index, first token, tokens) with at most ``max_step_tokens`` tokens
        each, entries in order, an entry that does not fit going on in the next chunk."""
        chunks, done = [], [0] * len(toks)
        while True:
            chunk, room = [], self.max_step_tokens
            for i, t in enumerate(toks):
                left = t.size - done[i]
                if left and room:
                    take = min(left, room, self.portion or room)
                    chunk.append((i, done[i], take))
                    room -= take
            if not chunk:
                return chunks
            chunks.append(chunk)
            for i, start, take in chunk:
                done[i] = start + take

    # ------------------------------------------------------------ the kernels' status word ----
    def _look_at_status(self, single_tokens: bool = False) -> None:
        """After every step: with ``check_kernels`` read the kernels' status word now, else start a copy of it. Single-token steps,
        whose products wait on barriers too (float32 runs, 9 to 64 sequences of large models), take turns: a copy costs some 20 us of
        the host's time, several hundredths of a short step, and one in ``STATUS_EVERY`` tells of all that came before."""
        if self.check_kernels:
            ops.gemm_tc_check(self.device)
            return
        self._steps_unseen = self._steps_unseen + 1 if single_tokens else self.STATUS_EVERY
        if self._steps_unseen >= self.STATUS_EVERY:
            self._steps_unseen = 0
            self._status_later()

    def _status_later(self) -> None:
        """Start a copy of the kernels' status word to pinned memory. It is looked at when the next step begins, without waiting for the
        device, and at ``check_status``; a bounded wait that gave up inside a kernel is then reported late instead of never: one
        step after a step of many tokens, ``STATUS_EVERY`` after one of single tokens."""
        status = ops.tc_status(self.device)
        if status is None:
            return
        if self._status_host is None:
            self._status_host = torch.zeros(1, dtype=torch.int32).pin_memory()
        elif self._status_event is not None and not self._status_event.query():
            return                      # the earlier copy has not landed yet; it will tell the same story
        self._status_host.copy_(status, non_blocking=True)
        self._status_event = torch.cuda.Event()
        self._status_event.record()

    def _raise_late_status(self, wait: bool = False) -> None:
        ev = self._status_event
        if ev is None or not (wait or ev.query()):
            return
        ev.synchronize()
        self._status_event = None
        if int(self._status_host[0]):
            ops.gemm_tc_check(self.device)          # reads the word itself, clears it and raises

    def check_status(self) -> None:
        """Raise if a kernel's bounded wait gave up in any step so far (waits for the device)."""
        self._raise_late_status(wait=True)
        ops.gemm_tc_check(self.device)

    # ------------------------------------------------------------------ chunks ----
    def _run_chunk(self, entries, slots, toks, chunk, out, out_base) -> None:
        book = self.cache.book
        c_slots = [slots[i] for i, _, _ in chunk]
        c_past = [int(book.lengths[s]) for s in c_slots]
        c_counts = [take for _, _, take in chunk]
        new_lens = [p + c for p, c in zip(c_past, c_counts)]
        book.grow(c_slots, new_lens)
        tokens = np.concatenate([toks[i][start:start + take] for i, start, take in chunk]).astype(np.int32)
        rows, dest = [], []
        base = 0
        for i, start, take in chunk:
            for j, w in enumerate(entries[i].want):
                w = int(w)
                if start <= w < start + take:
                    rows.append(base + w - start)
                    dest.append(out_base[i] + j)
            base += take
        order = np.argsort(np.asarray(dest, dtype=np.int64), kind="stable") if dest else np.zeros(0, dtype=np.int64)
        rows_a = np.asarray(rows, dtype=np.int32)[order] if rows else np.zeros(0, dtype=np.int32)
        dest_a = np.asarray(dest, dtype=np.int64)[order] if dest else np.zeros(0, dtype=np.int64)
        b = self.meta.upload(c_slots, c_past, c_counts, tokens, rows_a, book.tables_for(c_slots), seen=book.seen[c_slots] if book.budget else None)
        W = rows_a.shape[0]
        if self._chunk_by_graph(b, W, out, dest_a):
            pass
        elif W and np.array_equal(dest_a, np.arange(dest_a[0], dest_a[0] + W)):
            self.model.forward(b, self.cache, self.ws, out[int(dest_a[0]):int(dest_a[0]) + W])
        elif W:
            mark = self.ws.mark()
            tmp = self.ws.take((W, self.model.vocab), torch.float32)
            self.model.forward(b, self.cache, self.ws, tmp)
            out.index_copy_(0, torch.from_numpy(dest_a).to(self.device), tmp)
            self.ws.release(mark)
        else:
            self.model.forward(b, self.cache, self.ws, out[:0])
        book.commit(c_slots, new_lens)
        self._drop_drafts(c_slots, new_lens)

    def _chunk_by_graph(self, b, W: int, out, dest_a) -> bool:
        """A step of many tokens whose shape (tokens, sequences, longest share, wanted rows) has been seen before is
        recorded once as a CUDA graph and replayed from then on: the host then no longer issues some two hundred
        launches per step, which for short prompts is most of the step's time. Lengths, positions and tables live
        in the device buffer that the upload refreshed, so one recording serves every step of that shape. The logits
        land in a buffer of the stepper's and are copied to ``out``. Returns False if the step was not run."""
        most = self.max_graph_rows if b.tree is None else self.max_draft_rows
        if not (self.use_graphs and getattr(self.model, "capturable", True) and 0 < W <= most):
            return False
        self._check_graph_key()
        gkey = ("chunk" if b.tree is None else "drafts", b.T, b.n, b.max_count, W, b.fresh)      # parts may treat steps that start at position 0 differently
        graph = self._graphs.get(gkey)
        if graph is None and gkey not in self._seen_chunk:
            self._seen_chunk.add(gkey)
            if len(self._seen_chunk) > 4096:
                self._seen_chunk.clear()
            return False
        if self._chunk_logits is None or self._chunk_logits.shape[0] < W:
            self._chunk_logits = torch.empty((max(W, 8), self.model.vocab), dtype=torch.float32, device=self.device)
            for k in [k for k in self._graphs if isinstance(k[0], str)]:
                del self._graphs[k]
            graph = None
        logits = self._chunk_logits[:W]
        if graph is None:
            if sum(1 for k in self._graphs if isinstance(k[0], str)) >= self.max_chunk_graphs:
                for k in [k for k in self._graphs if isinstance(k[0], str)]:
                    del self._graphs[k]
            before = ops.lib().launches
            graph = self._graphs[gkey] = self._capture(b, logits)
            self._graph_own[gkey] = ops.lib().launches - before
            ops.lib().launches = before          # captured, not run
        graph.replay()
        self.graph_kernel_launches += self._graph_own[gkey]
        if np.array_equal(dest_a, np.arange(dest_a[0], dest_a[0] + W)):
            out[int(dest_a[0]):int(dest_a[0]) + W].copy_(logits)
        else:
            out.index_copy_(0, torch.from_numpy(dest_a).to(self.device), logits)
        return True

    def _check_graph_key(self) -> None:
        """Recordings hold addresses of the workspace and of the metadata buffer: when either was replaced, they go."""
        key = (self.ws.generation, self.meta.generation)
        if key != self._graph_key:
            self._graphs.clear()
            self._graph_key = key

    # ------------------------------------------------------------------ decode ----
    def _decode(self, entries, slots, toks, floats) -> torch.Tensor:
        tokens = np.asarray([int(t[0]) for t in toks], dtype=np.int32)
        logits = self._decode_core(slots, tokens, None, floats)
        n = len(slots)
        wanted = [i for i, e in enumerate(entries) if len(e.want)]
        if len(wanted) == n:
            return logits
        if not wanted:
            return logits[:0]
        return logits.index_select(0, torch.tensor(wanted, dtype=torch.long, device=self.device))

    def decode_fed(self, slots, feed_map) -> torch.Tensor:
        """One token for each of ``slots``, taken from the device-side feed: sequence i reads
        ``feed[feed_map[i]]``, where the sampler left the tokens it chose for the previous step's rows.
        Returns the logits of every row (a view that the next step overwrites)."""
        self._raise_late_status()
        book = self.cache.book
        slots = [int(s) for s in slots]
        if len(slots) > self.meta.FEED:
            raise ValueError(f"a device-fed step takes at most {self.meta.FEED} sequences")
        for s in slots:
            if int(book.seen[s]) + 1 > self.max_len:
                raise CacheFull(f"slot {s} would hold {int(book.seen[s]) + 1} tokens; the longest sequence allowed "
                                f"is {self.max_len}")
        return self._decode_core(slots, None, np.asarray(feed_map, dtype=np.int32), None)

    @property
    def feed(self) -> torch.Tensor:
        return self.meta.feed

    def _decode_core(self, slots, tokens, feed_map, floats) -> torch.Tensor:
        book = self.cache.book
        n = len(slots)
        past = [int(book.lengths[s]) for s in slots]
        new_lens = [p + 1 for p in past]
        book.grow(slots, new_lens)
        rows = np.arange(n, dtype=np.int32)
        if floats is None:
            floats = np.zeros(n, dtype=np.float32)
        b = self.meta.upload(slots, past, [1] * n, tokens, rows, book.tables_for(slots), floats=floats,
                             feed_map=feed_map, seen=book.seen[slots] if book.budget else None)
        self.last_batch = b
        if self._decode_logits is None or self._decode_logits.shape[0] < n:
            cap = max(n, 8 if self._decode_logits is None else 2 * self._decode_logits.shape[0])
            self._decode_logits = torch.empty((cap, self.model.vocab), dtype=torch.float32, device=self.device)
            self._graphs.clear()
        logits = self._decode_logits[:n]

        self._check_graph_key()
        gkey = (n, b.ids_map is not None)
        graph = self._graphs.get(gkey)
        if graph is not None:
            graph.replay()
            self.graph_kernel_launches += self._graph_own[gkey]
        elif (self.use_graphs and getattr(self.model, "capturable", True) and n <= self.max_graph_batch
              and gkey in self._seen_decode):
            before = ops.lib().launches
            self._graphs[gkey] = self._capture(b, logits)
            self._graph_own[gkey] = ops.lib().launches - before
            ops.lib().launches = before          # captured, not run
            self._graphs[gkey].replay()
            self.graph_kernel_launches += self._graph_own[gkey]
        else:
            self.model.forward(b, self.cache, self.ws, logits)
            self._seen_decode.add(gkey)
        book.commit(slots, new_lens)
        self._drop_drafts(slots, new_lens)
        self._look_at_status(single_tokens=True)
        return logits

    def _capture(self, b, logits):
        torch.cuda.synchronize(self.device)
        g = torch.cuda.CUDAGraph()
        self.ws.frozen = True
        try:
            with torch.cuda.graph(g):
                self.model.forward(b, self.cache, self.ws, logits)
        finally:
            self.ws.frozen = False
        return g
