"""Where drafted tokens come from.

A drafter is a callable: ids so far -> (tokens, parents), tokens that may follow them as a tree; ``parents[i]`` is the place of
the token that token i follows, before i (-1: the last id).  ``Engine.greedy`` runs them through the model in one step and keeps
those the model would have chosen.
"""
from __future__ import annotations

from typing import List, Sequence, Tuple


class PromptLookup:
    """What followed the last few ids where they stood before: the continuations of up to ``width`` earlier places of the last ``ngram`` ids (of
    fewer, where those are new), the latest first, up to ``depth`` tokens each, joined where they begin alike."""

    def __init__(self, ngram: int = 3, width: int = 4, depth: int = 8):
        if min(ngram, width, depth) < 1:
            raise ValueError("ngram, width and depth must be at least 1")
        self.ngram, self.width, self.depth = ngram, width, depth

    def __call__(self, ids: Sequence[int]) -> Tuple[List[int], List[int]]:
        ids = list(ids)
        tokens: List[int] = []
        parents: List[int] = []
        children = {}               # (place, token) -> the place of that child
        for n in range(min(self.ngram, len(ids) - 1), 0, -1):
            last, found = ids[-n:], 0
            for at in range(len(ids) - n - 1, -1, -1):
                if ids[at:at + n] != last:
                    continue
                place = -1
                for t in ids[at + n:at + n + self.depth]:
                    if (place, t) not in children:
                        children[place, t] = len(tokens)
                        tokens.append(t)
                        parents.append(place)
                    place = children[place, t]
                found += 1
                if found == self.width:
                    break
            if found:
                break
        return tokens, parents
