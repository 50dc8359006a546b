"""Guesses for what a sequence goes on with, for ``Engine(drafter=...)``.

A drafter is called with a sequence's tokens (prompt and output) and returns guesses as (tokens, parents): a tree, a guess's parent given by its place among
the guesses, -1 for those that would follow the last token itself; parents come before their children.  No guesses: ([], [])."""
from __future__ import annotations

from typing import Dict, List, Sequence, Tuple


class PromptLookup:
    """What followed the last tokens where they stood before: texts repeat themselves, and answers repeat their questions.

    The longest front of up to ``match`` last tokens that occurs earlier counts first, later occurrences before earlier ones; the ``length`` tokens behind each of
    up to ``branches`` occurrences make a tree of at most ``size`` guesses (common beginnings once).  Looks at the last ``window`` tokens."""

    def __init__(self, size: int = 12, length: int = 6, branches: int = 3, match: int = 3, window: int = 4096):
        if min(size, length, branches, match, window) <= 0:
            raise ValueError("PromptLookup: size, length, branches, match and window are 1 or more")
        self.size, self.length, self.branches, self.match, self.window = size, length, branches, match, window

    def __call__(self, tokens: Sequence[int]) -> Tuple[List[int], List[int]]:
        tokens = list(tokens[-self.window:])
        n, found = len(tokens), []
        places = [i for i in range(n - 2, -1, -1) if tokens[i] == tokens[-1]] if n > 1 else []
        for m in range(self.match, 0, -1):
            for i in places:
                if len(found) == self.branches:
                    break
                if i not in found and i >= m - 1 and tokens[i - m + 1:i + 1] == tokens[n - m:]:
                    found.append(i)
        guesses: List[int] = []
        parents: List[int] = []
        children: Dict[Tuple[int, int], int] = {}
        for i in found:
            at = -1
            for t in tokens[i + 1:i + 1 + self.length]:
                child = children.get((at, t))
                if child is None:
                    if len(guesses) == self.size:
                        break
                    child = children[(at, t)] = len(guesses)
                    guesses.append(t)
                    parents.append(at)
                at = child
        return guesses, parents
