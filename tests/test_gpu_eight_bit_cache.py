"""The engine over a cache of eight bits, with drafted tokens, and its log probabilities.

Two bfloat16 runs of one computation that differ in kernels, order of sums and batch differ by their roundings: about a dozen of 2^-9 (root mean
square) a layer and as many for the head, 3 layers: sqrt(48) 2^-9 = 1.4 % of the logits' spread.  CLOSE is four times that.
(Keys and values have to be rounded once, from 32 bits, on both sides: rounded to bfloat16 first, one in 16 would lie halfway between two codes, and half
of those would take the other one.)"""
import math

import pytest
import torch

from tests import helpers as H
from tests.plain import llama_plain as P

pytestmark = pytest.mark.gpu
CLOSE = 4 * math.sqrt(48) * 2.0 ** -9
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    return {name: H.make_folder(tmp_path_factory.mktemp("eight" + name), H.TINY[name][0], H.TINY[name][1], dtype="bfloat16", sharpen=3.0) for name in "ABC"}


def runner_of(folder, cache_dtype, n_pages=24, **kw):
    from lgml_b200.engine import ModelRunner

    return ModelRunner.from_folder(folder, torch.bfloat16, n_pages=n_pages, max_slots=6, cache_dtype=cache_dtype, max_step_tokens=512, **kw)


def near(a, b, what=""):
    off = (a - b).pow(2).mean().sqrt() / b.pow(2).mean().sqrt()
    assert torch.isfinite(a).all() and off <= CLOSE, (what, float(off))


def rounded_writes(monkeypatch):
    """Every key and value that a bfloat16 cache gets is put through eight bits, in torch."""
    from lgml_b200 import ops
    from lgml_b200.parts import rope

    plain = ops.rope_kv_write

    def write(qkv, positions, seq_of_token, block_table, inv_freq, n_rot, pairing, k_pages, v_pages, H, G, D, *args, **kw):
        x = (qkv.data.double().sum(0) + (0 if qkv.bias is None else qkv.bias.double()) if isinstance(qkv, ops.Partials) else qkv.double()).view(-1, H + 2 * G, D)
        angle = positions.double()[:, None, None] * inv_freq.double().sum(0)[:n_rot // 2]
        assert pairing == "half" and n_rot == D
        one, two, c, s = x[:, H:H + G, :D // 2], x[:, H:H + G, D // 2:], angle.cos(), angle.sin()
        sides = (torch.cat([one * c - two * s, one * s + two * c], -1), x[:, H + G:].clone())
        q = plain(qkv, positions, seq_of_token, block_table, inv_freq, n_rot, pairing, k_pages, v_pages, H, G, D, *args, **kw)
        p = positions.long()
        page = block_table.long()[seq_of_token.long(), p // 64]
        for pool, y in zip((k_pages, v_pages), sides):
            y = y.float()
            m, e = torch.frexp(y.abs().amax(-1, keepdim=True))
            step = ((torch.where(m <= 0.875, e - 9, e - 8).clamp(-60, 119) + 127).int() << 23).view(torch.float32)
            pool[page, :, p % 64] = ((y / step).to(E4M3).float() * step).to(torch.bfloat16)
        return q

    monkeypatch.setattr(rope.ops, "rope_kv_write", write)


def drive(runner, seqs):
    """Two prompts of several portions (one over 64 tokens beside a decoding request), then tokens one by one; all logits that were asked for."""
    got = []
    a, b = runner.open("a"), runner.open("b")
    A, B = seqs
    got.append(runner.step([(a, A[:30], [29])]))
    got.append(runner.step([(a, A[30:31], [0]), (b, B[:90], [0, 50, 89])]))
    got.append(runner.step([(a, A[31:101], [69]), (b, B[90:154], [63])]))
    for i in range(4):
        got.append(runner.step([(a, A[101 + i:102 + i], [0]), (b, B[154 + i:155 + i], [0])]).clone())         # (a replayed step's logits are its graph's buffer)
    got.append(runner.step([(b, B[158:225], list(range(67)))]))
    runner.rt.check_status()
    runner.close(a), runner.close(b)
    return torch.cat(got)


@pytest.mark.parametrize("name", ["B", "C"])
def test_logits_are_those_of_a_bfloat16_cache_whose_writes_are_rounded(folders, name, monkeypatch):
    vocab = H.TINY[name][0]["vocab_size"]
    seqs = [H.random_ids(110, vocab, 1), H.random_ids(230, vocab, 2)]
    eight = runner_of(folders[name], E4M3)
    got = [drive(eight, seqs), drive(eight, seqs)]          # (the second time, steps are replayed)
    plain = runner_of(folders[name], None)
    exact = drive(plain, seqs)
    assert eight.cache.bytes_held() < 0.57 * plain.cache.bytes_held()
    rounded_writes(monkeypatch)
    want = drive(runner_of(folders[name], None, use_graphs=False), seqs)
    for g in got:
        near(g, want, name)
    # and eight bits do show: the comparison above is of something
    assert (exact - want).pow(2).mean().sqrt() > 2.0 ** -9 * want.pow(2).mean().sqrt()


def test_generation_over_eight_bits_with_preemption_and_the_prefix_cache(folders):
    import lgml_b200

    folder = str(folders["B"])
    prompts = [H.random_ids(n, 320, 60 + n) for n in (5, 70, 131, 64)]
    wide = lgml_b200.Engine(folder, cache_dtype="float8_e4m3", slots=4, kv_tokens=2048)
    want = wide.generate(prompts, max_tokens=12, temperature=0.0)
    assert wide.runner.cache.page_dtype == E4M3
    tight = lgml_b200.Engine(folder, cache_dtype="fp8", slots=4, kv_tokens=320, prefix_cache=True)
    for _ in range(2):
        got = tight.generate(prompts, max_tokens=12, temperature=0.0)
        assert all(len(g) == 12 for g in got)
        for p, g in zip(prompts, got):
            consistent(wide, p, g)
    for p, g in zip(prompts, want):
        consistent(wide, p, g)


def consistent(eng, prompt, ids, slack=CLOSE):
    """Every id is the best of its logits, or so near to it that a rounding may have decided."""
    req = eng.runner.open(("check", id(ids)))
    try:
        logits = eng.runner.step([(req, list(prompt) + list(ids[:-1]), list(range(len(prompt) - 1, len(prompt) + len(ids) - 1)))])
    finally:
        eng.runner.close(req)
    spread = logits.std()
    for i, t in enumerate(ids):
        assert logits[i, t] >= logits[i].max() - 4 * slack * spread, (i, float(logits[i].max() - logits[i, t]), float(spread))


@pytest.mark.parametrize("cache_dtype", [None, E4M3])
@pytest.mark.parametrize("name", ["A", "B"])
def test_a_tree_of_drafted_tokens_has_the_logits_of_its_paths(folders, name, cache_dtype):
    """Two requests with trees in one step: every token's logits are those its path alone has; what is kept goes on, what is not is forgotten."""
    vocab = H.TINY[name][0]["vocab_size"]
    runner = runner_of(folders[name], cache_dtype)
    prefix = {"a": H.random_ids(61, vocab, 3), "b": H.random_ids(9, vocab, 4)}
    trees = {"a": (H.random_ids(12, vocab, 5), [-1, 0, 1, 1, 0, 2, 2, -1, 7, 3, 9, 10]), "b": (H.random_ids(3, vocab, 6), [-1, 0, 1])}
    live = {r: runner.open(r) for r in prefix}
    runner.step([(live[r], prefix[r], []) for r in prefix])

    def path(parents, i):
        return [] if i < 0 else path(parents, parents[i]) + [i]

    def alone(r, ids):
        req = runner.open(("alone", r))
        runner.step([(req, prefix[r], [])])
        out = [runner.step([(req, [t], [0])])[0].clone() for t in ids]
        runner.close(req)
        return out[-1]

    for _ in range(2):          # (the first tree is not kept)
        logits = runner.step_tree([(live[r], *trees[r]) for r in prefix])
        row = 0
        for r, (tokens, parents) in trees.items():
            for i in range(len(tokens)):
                near(logits[row], alone(r, [tokens[j] for j in path(parents, i)]), (r, i))
                row += 1
    runner.keep(live["a"], 3)
    runner.keep(live["b"], 0)
    assert live["a"].n_tokens == 64 and live["b"].n_tokens == 9
    more = runner.step([(live["a"], [7], [0]), (live["b"], [8], [0])]).clone()
    near(more[0], alone("a", trees["a"][0][:3] + [7]))
    near(more[1], alone("b", [8]))
    runner.rt.check_status()
    for r in live.values():
        runner.close(r)
    runner.cache.check()


@pytest.mark.parametrize("cache_dtype", [None, "float8_e4m3"])
def test_greedy_with_drafts_gives_what_the_argmax_gives(folders, cache_dtype):
    import lgml_b200
    from lgml_b200.engine.drafts import PromptLookup

    eng = lgml_b200.Engine(str(folders["B"]), cache_dtype=cache_dtype, slots=3, kv_tokens=1024)
    prompt = (H.random_ids(12, 320, 8) * 4)[:45]
    plain, t0 = eng.greedy(prompt, 60)

    def oracle(ids):            # the true continuation beside a wrong one, and so deep that it crosses pages
        at = len(ids) - len(prompt)
        right = plain[at:at + 9]
        return [5, *right, 3], [-1, -1, *range(1, len(right)), 0]

    def chain(ids):             # the same as a chain: its cells stay
        right = plain[len(ids) - len(prompt):][:20]
        return right, list(range(-1, len(right) - 1))

    for draft, most in ((PromptLookup(), 60), (oracle, 40), (chain, 40), (lambda ids: ([], []), 60), (lambda ids: (H.random_ids(63, 320, len(ids)), [-1] * 63), 60)):
        ids, t = eng.greedy(prompt, 60, draft=draft)
        assert len(ids) == 60 and t["steps"] <= most
        consistent(eng, prompt, ids)
        if ids == plain and draft in (oracle, chain):
            assert t["steps"] <= 14
    stop = plain[20]
    ids, _ = eng.greedy(prompt, 60, stop=[stop], draft=chain)
    assert ids[-1] == stop and stop not in ids[:-1] or stop not in ids
    assert not eng.runner.cache.live and eng.runner.cache.n_free_pages == eng.runner.cache.n_pages


def test_scores_of_given_and_of_generated_tokens(tmp_path):
    """In float32 against the plain implementation's log softmax in 64 bits: logits of this engine are within 2e-4 there (its replay tests), a difference of
    two of them and a logarithm of a mean of them within twice that."""
    import lgml_b200

    folder = H.make_folder(tmp_path, H.TINY_B, 1, dtype="float32")
    eng = lgml_b200.Engine(str(folder), dtype="float32", slots=2, ubatch=50)
    prompts = [H.random_ids(n, 320, n) for n in (1, 2, 51, 101, 130)]
    scored = eng.score(prompts, top=4)
    assert [len(s) for s in scored] == [0, 1, 50, 100, 129]

    def check(ids, first, scores, top):
        logs = torch.log_softmax(H.oracle_logits(folder, ids), -1)
        for i, sc in enumerate(scores, first):
            row = logs[i - 1]
            assert sc.id == ids[i] and abs(sc.logprob - row[ids[i]]) <= 5e-4
            assert abs(sc.entropy + (row.exp() * row).sum()) <= 2e-3
            order = torch.argsort(row, descending=True)
            assert len(sc.top) == top and all(abs(lp - row[t]) <= 5e-4 and lp >= float(row[order[j]]) - 1e-3 for j, (t, lp) in enumerate(sc.top))
            assert abs(float(row[order[sc.rank]] - row[ids[i]])) <= 1e-3

    for p, s in zip(prompts, scored):
        check(p, 1, s, 4)
    for opts in (dict(temperature=0.0), dict(temperature=1.0, seed=3, top_k=0, top_p=1.0, min_p=0.0), dict(temperature=0.7, seed=4, top_k=20), dict(temperature=0.7, seed=5, top_k=0, top_p=0.9)):
        for (ids, scores), p in zip(eng.generate(prompts[1:3], max_tokens=9, logprobs=3, **opts), prompts[1:3]):
            assert len(ids) == len(scores) == 9
            check(p + ids, len(p), scores, 3)
    assert eng.generate(prompts[1:2], max_tokens=2, temperature=0.0) == [eng.generate(prompts[1:2], max_tokens=2, temperature=0.0, logprobs=0)[0][0]]


def test_refusals(folders, tmp_path):
    import lgml_b200
    from lgml_b200.config import config_from_dict
    from lgml_b200.engine import ModelRunner
    from lgml_b200.engine.runner import StepError
    from tests.nelosun_helpers import CONFIGS

    folder = str(folders["B"])
    for kw in (dict(dtype="float32", cache_dtype="float8_e4m3"), dict(cache_dtype="float32"), dict(cache_dtype="int8")):
        with pytest.raises(ValueError):
            lgml_b200.Engine(folder, **kw)
    cfg = config_from_dict(CONFIGS["odd"])
    with pytest.raises(ValueError):
        ModelRunner.from_config(cfg, 0, torch.bfloat16, n_pages=8, cache_dtype=E4M3)
    runner = runner_of(folder, E4M3, n_pages=4)
    r = runner.open("r")
    for entry in ((r, [1, 2], [-1]), (r, [1, 2], [-1, 1]), (r, [1, 2], [-2, 0]), (r, [1] * 65, list(range(-1, 64))), (r, [1, 320], [-1, 0]), (r, [], [])):
        with pytest.raises(StepError):
            runner.step_tree([entry])
    with pytest.raises(StepError):
        runner.keep(r, 0)
    runner.step_tree([(r, [1, 2, 3], [-1, -1, 0])])
    for n in (2, 4, -1):
        with pytest.raises(StepError):
            runner.keep(r, n)
    runner.keep(r, 1)
    with pytest.raises(StepError):
        runner.keep(r, 0)
    runner.step_tree([(r, [1], [-1])])
    runner.step([(r, [4], [0])])
    with pytest.raises(StepError):
        runner.keep(r, 1)
    eng = lgml_b200.Engine(folder, slots=1)
    for call in (lambda: eng.score([[1, 2]], top=33), lambda: eng.score([[]]), lambda: eng.score([[1, 320]]), lambda: eng.score([[1] * 300]), lambda: eng.generate([[1]], logprobs=33)):
        with pytest.raises(ValueError):
            call()
