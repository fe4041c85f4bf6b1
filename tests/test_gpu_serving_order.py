"""Kernels that start ahead of one another's end: what stands between a kernel and one that reads its results."""
import pytest
import torch

from tests.test_gpu_serving_ops import Problem, ints, status

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads", [(8, 2, 64), (32, 2, 64)])
def test_an_attention_call_without_a_request_in_range_keeps_the_order(heads):
    """A kernel that takes its time and lets the next start at once, an attention call none of whose requests is between the two lengths, a kernel that reads
    what the first wrote (in memory where other numbers stood before)."""
    from lgml_b200 import ops

    H, G, D = heads
    p = Problem([3, 2], [100, 70], H, G, D, True)
    out = torch.full_like(p.q, 7.0)
    st = status()
    top = 32
    inputs = [torch.randn(300, 60000, device=p.q.device, generator=torch.Generator(p.q.device).manual_seed(i)) for i in range(2)]
    ids = ints([0] * 300)
    args = (p.q, ints(p.positions), ints(p.start), ints(p.pos0), ints(p.table), p.k, p.v, out, H, p.scale, 0, st, 9, 103)
    for turn in range(20):
        x = inputs[turn % 2]
        first = ops.token_logprobs(x, ids, top, st)
        ops.tree_attention(*args, k_exps=p.ke, v_exps=p.ve, min_new_tokens=5)
        second = ops.token_logprobs(first.top_logprobs, ids, 4, st)
        torch.cuda.synchronize()
        again = ops.token_logprobs(first.top_logprobs, ids, 4, st)
        assert all(torch.equal(a, b) for a, b in zip(second, again))
        del first, second, again
    assert st.item() == 0 and (out == 7.0).all()
