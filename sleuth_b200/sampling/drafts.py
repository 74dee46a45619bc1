"""Drafting: tokens that a sequence may go on with, looked up in its own text, judged several at a time in one step.

``DraftPolicy(tokens=8)``: before each step the latest tokens of a sequence are looked for further up in its text (the longest phrase
of up to ``ngram`` tokens that occurs there), and what followed it then is drafted: up to ``tokens`` tokens, with ``branches`` > 1 as a
tree of the continuations of several occurrences. One step then runs the newest token and all drafts; every draft
that is the token which would have been chosen anyway is one step less. The choices are made as without drafts, random ones too (a token's
random number belongs to its place in the text, not to the step), from logits of a step of several tokens: in float32 its sums differ from a single token's in their
last bits, in bfloat16 its products and its attention round otherwise, so choices between near-equal logits may differ, and the text behind them.

Nothing here touches a GPU; the loop that uses it is ``engine/generate.py``, the step ``engine/stepper.py``. A text that
repeats itself (code, tables, quotations) gains, another one pays a wider step for little.
"""

from __future__ import annotations

from dataclasses import dataclass


@dataclass(frozen=True)
class DraftPolicy:
    tokens: int = 8             # drafted tokens of a sequence in a step, at most
    branches: int = 1           # continuations that a step tries
    ngram: int = 3              # the longest phrase that is looked for

    def __post_init__(self):
        for name, most in (("tokens", 255), ("branches", 255), ("ngram", 64)):
            v = getattr(self, name)
            if not isinstance(v, int) or isinstance(v, bool) or not 1 <= v <= most:
                raise ValueError(f"drafts: {name} must be a whole number from 1 to {most}, got {v!r}")


class NgramDrafter:
    """The text of one sequence and where its phrases occurred. A phrase is kept with the places behind its latest occurrences,
    so a token costs ``ngram`` dictionary steps and a lookup as many."""

    def __init__(self, policy: DraftPolicy, ids=()):
        self.policy = policy
        self.text: list[int] = []
        self._behind: dict[tuple, list[int]] = {}
        for t in ids:
            self.add(t)

    def add(self, token: int) -> None:
        # what ends at the last token is followed by this one
        end = len(self.text)
        for n in range(1, min(self.policy.ngram, end) + 1):
            places = self._behind.setdefault(tuple(self.text[end - n:end]), [])
            places.append(end)
            if len(places) > 2 * self.policy.branches:
                del places[0]
        self.text.append(int(token))

    def propose(self, room: int) -> tuple[list[int], list[int]]:
        """Up to ``room`` drafted tokens and, for each, the node that it continues: 0 for the text's last token, i for the i-th draft."""
        room = min(room, self.policy.tokens)
        tokens: list[int] = []
        parents: list[int] = []
        if room <= 0:
            return tokens, parents
        end = len(self.text)
        for n in range(min(self.policy.ngram, end), 0, -1):
            places = self._behind.get(tuple(self.text[end - n:]))
            if places:
                break
        else:
            return tokens, parents
        children: dict[tuple[int, int], int] = {}
        tried = 0
        for place in reversed(places):
            if tried == self.policy.branches or len(tokens) == room:
                break
            node, fresh = 0, False
            for token in self.text[place:place + room]:
                child = children.get((node, token))
                if child is None:
                    if len(tokens) == room:
                        break
                    tokens.append(token)
                    parents.append(node)
                    child = children[node, token] = len(tokens)
                    fresh = True
                node = child
            tried += fresh
        return tokens, parents
