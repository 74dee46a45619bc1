"""What a cache of bounded size keeps, for texts longer than it.

``KeepPolicy(window=w, first=f)``: every query sees the latest ``w`` tokens and the first ``f`` ones, and the pages between them are
given back (attention with a sliding window and first tokens that stay visible).

``KeepPolicy(budget=B, first=f, recent=r)``: a query sees all that its layer still holds. After every step each key/value head of each
layer keeps at most ``B`` tokens of a sequence: the first ``f``, the latest ``r`` (half of ``B`` when not given) and, of the others, those to
which the queries so far have given the largest sum of softmax weights. A prompt goes in portions of ``portion`` tokens, with an
eviction after each, so a sequence never holds more than ``B + portion`` rows, nor more than the longest text has tokens. Tokens keep the rotation
of their own position. Beside the cache's pages every slot (``max_sequences``) takes 8 bytes a row, key/value head and layer for what its rows have
gathered and their positions; the number of slots goes by the pages when none is named, so a program that knows how many texts it serves at once names it.

``Engine.from_pretrained(folder, keep=KeepPolicy(...))``, ``sleuth_b200.load(folder, keep=...)`` or ``generate --keep-window/--keep-budget``.
"""

from __future__ import annotations

from dataclasses import dataclass


@dataclass(frozen=True)
class KeepPolicy:
    budget: int = 0             # rows that stay after a step for each key/value head (0: no eviction)
    window: int = 0             # latest tokens that a query sees, its own included (0: no window)
    first: int = 4              # first tokens that stay
    recent: int | None = None   # latest tokens that stay under a budget (None: half of the budget)
    portion: int = 512          # tokens of one sequence in a step under a budget

    def __post_init__(self):
        for name in ("budget", "window", "first", "portion"):
            v = getattr(self, name)
            if not isinstance(v, int) or isinstance(v, bool) or v < 0:
                raise ValueError(f"keep: {name} must be a whole number, not negative, got {v!r}")
            if v >= 1 << 31:
                raise ValueError(f"keep: {name} must be below 2^31, got {v}")
        if (self.budget > 0) == (self.window > 0):
            raise ValueError(f"keep: give a budget or a window, one of them (budget {self.budget}, window {self.window})")
        if self.recent is not None and (not isinstance(self.recent, int) or isinstance(self.recent, bool) or self.recent < 0):
            raise ValueError(f"keep: recent must be a whole number, not negative, got {self.recent!r}")
        if self.window and self.recent is not None:
            raise ValueError("keep: recent goes with a budget; under a window the window says how many latest tokens are seen")
        if self.budget and self.first + self.latest > self.budget:
            raise ValueError(f"keep: {self.first} first and {self.latest} recent tokens do not fit a budget of {self.budget}")
        if self.budget and self.portion < 1:
            raise ValueError("keep: a portion holds at least one token")

    @property
    def latest(self) -> int:
        """The latest tokens that an eviction leaves."""
        return min(self.budget // 2, max(0, self.budget - self.first)) if self.recent is None else self.recent

    @property
    def most_rows(self) -> int:
        """Rows that a sequence holds at most under a budget."""
        return self.budget + self.portion

    def rows_for(self, longest: int) -> int:
        """The same where no text is longer than ``longest`` tokens."""
        return min(self.most_rows, longest)
