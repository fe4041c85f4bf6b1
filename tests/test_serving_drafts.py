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


def cached(monkeypatch, lens, calls, visible=None, group=4, dim=64):
    """The calls of ``tree_attention`` that ``cached_attention`` makes for requests that bring these numbers of tokens, over e4m3 pages of two KV heads."""
    from types import SimpleNamespace

    from lgml_b200 import ops

    monkeypatch.setattr(ops, "sm_count", lambda: 148)
    monkeypatch.setattr(ops, "tree_attention", lambda *a, **kw: calls.append(kw))
    H, G, N = 2 * group, 2, sum(lens)
    q = torch.zeros(N, H * dim, dtype=torch.bfloat16)
    pages = torch.zeros(1, G, 64, dim, dtype=torch.uint8).view(torch.float8_e4m3fn)
    exps = torch.zeros(1, G, 64, dtype=torch.uint8)
    batch = SimpleNamespace(positions=None, seq_start=None, seq_pos0=None, seq_lens=lens, max_kv_len=4000, max_q_len=max(lens), visible=visible)
    cache = SimpleNamespace(block_table=None, k=pages, v=pages, k_exps=exps, v_exps=exps)
    ops.cached_attention(q, batch, cache, torch.empty_like(q), H, 0.1, 0, None)
    return calls


@pytest.mark.parametrize("tokens,tall", [(5, False), (8, False), (9, True), (64, True)])
def test_ranges_are_planned_for_the_kernel_that_runs(monkeypatch, tokens, tall):
    """Many decoded tokens beside portions of 17 to 32 rows a KV head, which e4m3 pages of more KV heads than SMs leave to the few rows' kernel, and of more."""
    from lgml_b200 import ops

    first, second = cached(monkeypatch, [1] * 80 + [tokens] * 20, [])
    assert (first["max_new_tokens"], first["min_new_tokens"], second["max_new_tokens"], second["min_new_tokens"]) == (1, 1, tokens, 2)
    cuts = {t: ops.tree_splits(20, 2, 4 * tokens, 4000, 64, tall=t) for t in (False, True)}
    assert second["n_splits"] == cuts[tall] and (tall or cuts[True] != cuts[False])


def test_a_tree_of_too_many_tokens_is_refused_before_anything_is_launched(monkeypatch):
    from lgml_b200 import ops

    calls = []
    with pytest.raises(ops.KernelError, match="64 tokens"):
        cached(monkeypatch, [3, 65], calls, visible=object())
    assert not calls and len(cached(monkeypatch, [3, 64], calls, visible=object())) == 1
