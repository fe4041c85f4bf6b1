"""The cache of eight bits, drafted tokens and log probabilities, as far as they need no GPU: what the C entries refuse before they launch, the cache's
books, the description of a tree step, the drafter."""
import ctypes
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from lgml_b200 import csrc
from lgml_b200.cache import CacheManager, FixedState, PagedKV
from lgml_b200.engine.batch import StepBatch, cache_view_of
from lgml_b200.engine.drafts import PromptLookup

P, F, L = ctypes.c_void_p, ctypes.c_float, ctypes.c_longlong
E4M3 = torch.float8_e4m3fn


def refused(library, symbol, args, what):
    lib = csrc.load(library)
    rc = getattr(lib, symbol)(*args)
    err = getattr(lib, f"lgml_{library}_last_error")
    err.restype = ctypes.c_char_p
    assert rc == -1 and what in err().decode(), (rc, err().decode())


def at(*pairs, size):
    """Arguments that are all fine (a pointer that nobody reads for None), with some replaced."""
    out = list(size)
    for i, v in pairs:
        out[i] = v
    return out


def test_store_and_read_refuse_before_a_launch():
    p = P(0x1000)
    good = [p, 1, 384, 1, L(0), None, p, 256, p, None, p, p, 2, 4, p, p, 64, 0, p, p, p, p, 9, 64, 5, 4, 1, 64, 1, p, None]
    for change, what in (((23, 32), "pages of 32"), ((27, 24), "head_dim 24"), ((27, 272), "head_dim 272"), ((16, 63), "n_rot 63"), ((16, 66), "n_rot 66"), ((16, -2), "n_rot"),
                         ((20, None), "exponents"), ((3, 0), "bad sizes"), ((25, 0), "bad sizes"), ((1, 7), "element type 7"), ((26, 300000), "too many heads")):
        refused("kv_store", "lgml_rope_kv_store", at(change, size=good), what)
    good = [p, p, p, p, 9, 64, p, 3, p, p, 2, 64, p, None]
    for change, what in (((5, 16), "pages of 16"), ((11, 20), "head_dim 20"), ((0, P(0x1008)), "aligned"), ((10, 0), "bad sizes"), ((7, 1 << 30), "too many")):
        refused("kv_store", "lgml_kv_read", at(change, size=good), what)


@pytest.mark.parametrize("library,symbol", [("attention_tree", "lgml_tree_attention"), ("attention_tree_tall", "lgml_tree_attention_tall")])
def test_attention_refuses_before_a_launch(library, symbol):
    p = P(0x1000)
    good = [p, 512, p, p, p, None, p, 2, 4, p, p, p, p, 9, 64, p, 512, p, 1, 5, 1, 4, 8, 2, 64, F(0.1), 0, p, None]
    for change, what in (((14, 128), "pages of 128"), ((22, 7), "no multiple"), ((24, 40), "head_dim 40"), ((21, 0), "new tokens"), ((21, 65), "new tokens"), ((20, 0), "new tokens"), ((20, 5), "new tokens"), ((18, 0), "ranges"),
                         ((18, 257), "ranges"), ((11, None), "exponents"), ((9, P(0x1008)), "aligned"), ((1, 511), "aligned"), ((7, 1 << 30), "too many requests")):
        refused(library, symbol, at(change, size=good), what)
    refused(library, symbol, at((18, 9), (17, None), size=good), "scratch")


def test_logprobs_refuse_before_a_launch():
    p = P(0x1000)
    good = [p, L(100), 3, 100, p, 5, 1, p, p, p, p, p, p, None]
    for change, what in (((3, 0), "0 logits"), ((1, L(99)), "99 apart"), ((5, 33), "33 alternatives"), ((5, -1), "alternatives"), ((3, (1 << 30) + 1), "apart"), ((6, 3), "slices"), ((6, 32), "slices"),
                         ((0, P(0x1002)), "off 4 bytes")):
        refused("logprobs", "lgml_token_logprobs", at(change, size=good), what)
    refused("logprobs", "lgml_token_logprobs", at((3, 4), (5, 5), (1, L(4)), size=good), "alternatives")
    slices = csrc.load("logprobs").lgml_token_logprobs_slices
    for n, v in ((0, 5), (1, 1), (1, 128256), (8, 128256), (1021, 128256), (1, 1 << 30), (100000, 32000)):
        s = slices(n, v, 148)
        assert 1 <= s <= 16 and s & (s - 1) == 0 and (s == 1 or s <= (v + 3 + 4095) // 4096)


def test_a_cache_of_eight_bits_keeps_codes_and_exponents():
    cm = CacheManager({0: PagedKV(2, 32), 1: PagedKV(2, 32), 2: PagedKV(2, 32, window=64)}, n_pages=5, max_slots=2, dtype=torch.bfloat16, device="cpu", page_dtype=E4M3)
    for g in cm.groups:
        for layer in g.layers:
            assert g.k[layer].dtype == g.v[layer].dtype == E4M3 and g.k_exps[layer].shape == g.k[layer].shape[:3] and g.v_exps[layer].dtype == torch.uint8
    assert cm.bytes_held() == sum(2 * g.pool.n_pages * 2 * 64 * (32 + 1) * len(g.layers) for g in cm.groups)
    view = cache_view_of(cm, 2, [torch.zeros(1, 1)] * 2)
    assert view.group == 1 and view.k_exps is cm.groups[1].k_exps[2]
    assert cache_view_of(CacheManager({0: PagedKV(2, 32)}, 5, 2, torch.bfloat16, "cpu"), 0, [None]).k_exps is None
    for spec in (PagedKV(2, 32, v_head_dim=16), PagedKV(2, 32, v_heads=1), PagedKV(2, 32, v_head_dim=16, v_in_k=True)):
        with pytest.raises(ValueError):
            CacheManager({0: spec}, n_pages=5, max_slots=2, dtype=torch.bfloat16, device="cpu", page_dtype=E4M3)


def test_a_tree_steps_description():
    cm = CacheManager({0: PagedKV(1, 32), 1: FixedState((3,))}, n_pages=8, max_slots=3, dtype=torch.bfloat16, device="cpu")
    a, b = cm.open("a"), cm.open("b")
    for r, n in ((a, 70), (b, 3)):
        cm.reserve(r, n), cm.commit(r, n)
    cm.reserve(a, 64), cm.reserve(b, 2)
    parents = [[-1, 0, 0, -1, 3] + list(range(4, 63)), [-1, -1]]
    batch = StepBatch(cm, [a, b], [[1] * 64, [2, 3]], [range(64), range(2)], "cpu")
    assert batch.cells is None and batch.visible is None
    batch.tree(parents)
    assert batch.cells.tolist() == list(range(70, 134)) + [3, 4]
    assert batch.positions.tolist() == [70, 71, 71, 70, 71] + [72 + i for i in range(59)] + [3, 3]
    masks = [m & (1 << 64) - 1 for m in batch.visible.tolist()]
    assert masks[:5] == [1, 3, 5, 8, 24] and masks[63] == sum(1 << i for i in range(3, 64)) and masks[64:] == [1, 2]
    # pages to read back: of the long request's, each once; entries of the others are none
    pages, table = batch.read_back(0, 10)
    assert pages.tolist() == a.tables[0] and table.tolist() == [[0, 1, 2], [-1, -1, -1]]
    b.tables[0][0] = a.tables[0][1]           # (as the prefix cache shares them)
    shared = StepBatch(cm, [a, b], [[1] * 64, [2, 3]], [range(64), range(2)], "cpu")
    pages, table = shared.read_back(0, 1)
    assert pages.tolist() == a.tables[0] and table.tolist() == [[0, 1, 2], [1, -1, -1]]
    assert shared.read_back(0, 1)[0] is pages


def test_prompt_lookup():
    look = PromptLookup(ngram=2, width=3, depth=3)
    assert look([1]) == ([], []) and look([1, 2, 3]) == ([], [])
    # the latest place first, joined where the continuations begin alike, none longer than the depth
    ids = [7, 8, 1, 2, 3, 7, 8, 1, 4, 7, 8, 5, 7, 8]
    tokens, parents = look(ids)
    assert tokens == [5, 7, 8, 1, 4, 7, 2, 3] and parents == [-1, 0, 1, -1, 3, 4, 3, 6]
    # fewer ids where the last two are new together
    assert look([4, 9, 6, 5, 9]) == ([6, 5, 9], [-1, 0, 1])
    assert PromptLookup(ngram=1, width=1, depth=2)(np.array([3, 1, 2, 3])) == ([1, 2], [-1, 0])
    for kw in (dict(ngram=0), dict(width=0), dict(depth=0)):
        with pytest.raises(ValueError):
            PromptLookup(**kw)


def test_names_of_cache_types():
    from lgml_b200.engine.engine import parse_cache_dtype
    from lgml_b200.engine.runner import ModelRunner

    assert parse_cache_dtype(None) is None and parse_cache_dtype("fp8") is E4M3 and parse_cache_dtype("float8_e4m3") is E4M3 and parse_cache_dtype(torch.bfloat16) is torch.bfloat16
    with pytest.raises(ValueError):
        parse_cache_dtype("int8")
    with pytest.raises(ValueError, match="bfloat16"):
        ModelRunner(SimpleNamespace(takes_trees=True), SimpleNamespace(dtype=torch.float32), n_pages=2, cache_dtype=E4M3)
    with pytest.raises(ValueError, match="plain attention"):
        ModelRunner(SimpleNamespace(takes_trees=False), SimpleNamespace(dtype=torch.bfloat16), n_pages=2, cache_dtype=E4M3)
