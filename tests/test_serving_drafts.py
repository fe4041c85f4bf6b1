"""Drafted tokens as far as they need no GPU: the room they may take, and which of them a call still wants."""
import numpy as np
import pytest
import torch

from lgml_b200.cache import CacheManager, PagedKV
from lgml_b200.engine.engine import Engine
from lgml_b200.engine.runner import StepError


def test_cells_that_a_request_can_still_have():
    cm = CacheManager({0: PagedKV(1, 32), 1: PagedKV(1, 32, window=100)}, n_pages=5, max_slots=2, dtype=torch.bfloat16, device="cpu", max_step_tokens=64)
    a, b = cm.open("a"), cm.open("b")
    held = {a: 0, b: 0}
    for req, n in ((a, 70), (b, 1), (a, 64), (b, 60), (a, 30), (a, 1)):
        left = cm.cells_left(req)
        if cm.reserve(req, n):
            assert n <= left
            cm.commit(req, n)
            held[req] += n
        else:
            assert n > left
        for r in (a, b):
            left = cm.cells_left(r)
            lens = [len(t) for t in r.tables]
            assert not cm.reserve(r, left + 1) and cm.reserve(r, left)
            cm.unreserve(r, lens)
    assert held[a] > 128


def test_drafts_that_lie_too_deep_are_left_out():
    tokens, parents = [5, 6, 7, 8, 9, 10], [-1, 0, 1, 0, -1, 4]
    draft = lambda ids: (tokens, parents)  # noqa: E731
    assert Engine._drafts(draft, [1], 9) == (tokens, parents)
    assert Engine._drafts(draft, [1], 3) == ([5, 6, 8, 9, 10], [-1, 0, 0, -1, 3])
    assert Engine._drafts(draft, [1], 2) == ([5, 9], [-1, -1])
    assert Engine._drafts(draft, [1], 1) == ([], [])
    assert Engine._drafts(lambda ids: (np.array([3, 4]), np.array([-1, 0])), [1], 5) == ([3, 4], [-1, 0])
    for bad in (([1, 2], [-1]), ([1, 2], [0, -1]), ([1, 2], [-1, 1])):
        with pytest.raises(StepError):
            Engine._drafts(lambda ids: bad, [1], 5)
