"""Drafted tokens from a sequence's own text: what followed the last time the same tokens stood there.

A `Lookup` remembers, for every run of one to three tokens of its sequence, where the run last ended. A tree of drafted tokens
takes the continuations of the places that the sequence's last tokens came from, the longest run first, and lays those that begin
alike over one another. Nothing is learned and nothing is read but the sequence; text that repeats itself (code, tables, quoted
passages) is drafted well, other text costs a step of a few more rows.
"""
from __future__ import annotations

from typing import Sequence

LONGEST = 3                # tokens of a run
PLACES = 2                 # places remembered for a run


class Lookup:
    def __init__(self, tokens: Sequence[int] = ()):
        self.tokens: list[int] = []
        self._ends: dict[tuple, list[int]] = {}    # run -> the last places behind it (index of the token that followed)
        self.extend(tokens)

    def extend(self, tokens: Sequence[int]) -> None:
        for t in tokens:
            at = len(self.tokens)
            for n in range(1, min(LONGEST, at) + 1):
                ends = self._ends.setdefault(tuple(self.tokens[at - n:at]), [])
                ends.append(at)
                del ends[:-PLACES]
            self.tokens.append(int(t))

    def tree(self, room: int) -> tuple[list[int], list[int]]:
        """(tokens, parents) of a tree of at most 1 + room rows, row 0 the sequence's last token."""
        tokens, parents = [self.tokens[-1]], [-1]
        n = len(self.tokens)
        for length in range(min(LONGEST, n), 0, -1):
            for place in reversed(self._ends.get(tuple(self.tokens[n - length:]), ())):
                at = 0
                for t in self.tokens[place:place + room]:
                    child = next((i for i in range(at + 1, len(tokens)) if parents[i] == at and tokens[i] == t), None)
                    if child is None:
                        if len(tokens) > room:
                            return tokens, parents
                        child = len(tokens)
                        tokens.append(t)
                        parents.append(at)
                    at = child
        return tokens, parents
