"""What the engine gives with log probabilities and with drafted tokens, where the plain calls of ``test_gpu_eight_bit_cache.py`` do not look."""
import math

import pytest
import torch

from tests import helpers as H

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    return H.make_folder(tmp_path_factory.mktemp("serving"), H.TINY_B, 1, dtype="float32")


EDITS = dict(repeat_penalty=1.4, frequency_penalty=0.3, presence_penalty=0.2, logit_bias={5: 6.0, 9: -4.0, 11: -math.inf, 17: 5.5})


@pytest.mark.parametrize("common,per_prompt", [
    (dict(temperature=0.0), None), (dict(temperature=0.8, seed=3, top_k=0, top_p=0.9), None), (dict(temperature=0.8, seed=4, top_k=200), None), (dict(temperature=0.8, seed=5, top_k=20), None),
    (dict(temperature=0.8, seed=6, **EDITS), [dict(top_k=20), dict(top_k=7), dict(temperature=0.0)])])
def test_scores_are_of_the_distribution_behind_bias_and_penalties(folder, common, per_prompt):
    """Logits of this engine in float32 are within 2e-4 of the plain implementation's; a penalty makes that 1.4 times as much, a difference of two of
    them twice that: 6e-4, and the entropy's weighted mean of log probabilities is as far off."""
    import lgml_b200

    eng = lgml_b200.Engine(str(folder), dtype="float32", slots=3)
    prompts = [H.random_ids(n, 320, n) for n in (3, 20, 9)]
    got = eng.generate(prompts, max_tokens=8, logprobs=4, per_prompt=per_prompt, **{**EDITS, **common})
    for p, (ids, scores) in zip(prompts, got):
        assert len(ids) == len(scores) == 8
        logits = H.oracle_logits(folder, p + ids).double()
        for i, sc in enumerate(scores):
            row = logits[len(p) + i - 1].clone()
            for t, b in EDITS["logit_bias"].items():
                row[t] += b
            for t in set(ids[:i]):
                row[t] = row[t] * 1.4 if row[t] <= 0 else row[t] / 1.4
                row[t] -= ids[:i].count(t) * 0.3 + 0.2
            logs = torch.log_softmax(row, -1)
            assert sc.id == ids[i] and abs(sc.logprob - logs[ids[i]]) <= 1e-3, (i, sc, float(logs[ids[i]]))
            weighted = torch.where(logs == -math.inf, torch.zeros_like(logs), logs.exp() * logs)
            assert abs(sc.entropy + weighted.sum()) <= 3e-3
            order = torch.argsort(row, descending=True)
            assert len(sc.top) == 4 and all(abs(lp - logs[t]) <= 1e-3 and lp >= float(logs[order[j]]) - 2e-3 for j, (t, lp) in enumerate(sc.top))
            assert abs(float(logs[order[sc.rank]] - logs[ids[i]])) <= 2e-3


@pytest.mark.parametrize("options", [dict(temperature=0.0), dict(temperature=0.8, seed=1, top_k=20), dict(temperature=0.8, seed=1, top_k=0, top_p=0.9)])
def test_a_status_that_the_scores_set_is_of_their_own_step(folder, options, monkeypatch):
    """The status word as the kernel would leave it after its copies' time ran out."""
    import lgml_b200
    from lgml_b200 import ops

    eng = lgml_b200.Engine(str(folder), dtype="float32", slots=1)
    plain = ops.token_logprobs

    def timed_out(logits, ids, top, status):
        got = plain(logits, ids, top, status)
        status.fill_(15)
        return got

    monkeypatch.setattr(ops, "token_logprobs", timed_out)
    with pytest.raises(RuntimeError, match="log probabilities"):
        eng.generate([[1, 2, 3]], max_tokens=1, logprobs=2, **options)
    assert eng.rt.status.item() == 0


@pytest.mark.parametrize("name", ["B", "C"])
@pytest.mark.parametrize("cache_dtype", [None, "float8_e4m3"])
def test_drafts_need_no_more_room_than_the_tokens(tmp_path, name, cache_dtype):
    """A pool of two pages that plain greedy decoding fills but for one cell, and drafters that would have more."""
    import lgml_b200
    from tests.test_gpu_eight_bit_cache import consistent

    config, seed = H.TINY[name]
    folder = H.make_folder(tmp_path, config, seed, dtype="bfloat16", sharpen=3.0)
    vocab = config["vocab_size"]
    eng = lgml_b200.Engine(str(folder), cache_dtype=cache_dtype, slots=1, kv_tokens=128)
    prompt = H.random_ids(45, vocab, 8)
    plain, _ = eng.greedy(prompt, 83)
    assert len(plain) == 83

    def right(ids):
        more = plain[len(ids) - len(prompt):][:30]
        return more + [1] * 20, [-1] + list(range(len(more) - 1)) + [-1] * 20 if more else [-1] * 20

    for draft in (right, lambda ids: (H.random_ids(63, vocab, len(ids)), [-1] * 63), lambda ids: (H.random_ids(63, vocab, len(ids)), list(range(-1, 62)))):
        got, t = eng.greedy(prompt, 83, draft=draft)
        assert len(got) == 83 and t["steps"] <= 82
        consistent(eng, prompt, got)
        assert not eng.runner.cache.live and eng.runner.cache.n_free_pages == eng.runner.cache.n_pages


def test_drafts_are_gone_once_another_step_may_have_written_over_them(tmp_path, monkeypatch):
    """A step of the request that fails in its layers, and one that is refused before anything runs."""
    from lgml_b200.engine import ModelRunner
    from lgml_b200.engine.runner import StepError

    folder = H.make_folder(tmp_path, H.TINY_B, 1, dtype="bfloat16")
    runner = ModelRunner.from_folder(folder, torch.bfloat16, n_pages=4, max_slots=2, max_step_tokens=64)
    a, b = runner.open("a"), runner.open("b")
    forward = runner.model.forward
    tree = [(a, [1, 2], [-1, 0]), (b, [3], [-1])]

    def broken(*args, **kw):
        forward(*args, **kw)
        raise RuntimeError("a layer failed")

    for fails in (lambda: runner.step([(a, [4, 5], [0])]), lambda: runner.step_tree([(a, [6], [-1])]),
                  lambda: runner.decode_step([a], torch.tensor([7], dtype=torch.int32, device=runner.rt.device))):
        runner.step_tree(tree)
        with monkeypatch.context() as m:
            m.setattr(runner.model, "forward", broken)
            with pytest.raises(RuntimeError, match="a layer failed"):
                fails()
        with pytest.raises(StepError, match="no drafted tokens"):
            runner.keep(a, 1)
    runner.step_tree(tree)
    with pytest.raises(StepError):
        runner.step([(a, [320], [0])])
    runner.step([(b, [9], [0])])
    runner.keep(a, 2)
    assert (a.n_tokens, b.n_tokens) == (2, 1)
    with pytest.raises(StepError):
        runner.keep(b, 1)
