"""What the sources of the serving kernels must keep to, seen without a GPU."""
import re

import pytest

from lgml_b200 import csrc


def end_of_block(source, at):
    """Where the block ends whose inside begins at ``at``."""
    depth = 1
    while depth:
        depth += {"{": 1, "}": -1}.get(source[at], 0)
        at += 1
    return at


def kernels(name):
    """The bodies of a file's kernels, without the functions inside them (whose returns leave those alone)."""
    source = re.sub(r"//[^\n]*", "", (csrc.HERE / name).read_text())
    for m in re.finditer(r"__global__[^{;]*?(\w+)\([^{;]*\)\s*{", source):
        body = source[m.end():end_of_block(source, m.end())]
        while inner := re.search(r"\[&\]\([^{;]*\)[^{;]*{", body):
            body = body[:inner.start()] + body[end_of_block(body, inner.end()):]
        yield m.group(1), body


@pytest.mark.parametrize("name", ["attention_tree.cu", "attention_tree_tall.cu", "tree_common.cuh", "logprobs.cu"])
def test_no_block_leaves_ahead_of_the_wait(name):
    """A grid whose blocks all leave without ``griddepcontrol.wait`` may be over before the kernel ahead of it is, and the kernel behind it waits for this
    grid alone."""
    found = list(kernels(name))
    assert found
    for kernel, body in found:
        main = body.rindex("pdl_wait();")
        for m in re.finditer(r"\breturn;", body[:main]):
            branch = body[body.rindex("{", 0, m.start()):m.start()]
            assert "pdl_wait();" in branch, (kernel, branch)


@pytest.mark.parametrize("name", ["attention_tree.cu", "attention_tree_tall.cu", "logprobs.cu"])
def test_warps_come_together_ahead_of_a_cluster_barrier(name):
    """``barrier.cluster`` is ``.aligned``: all threads of a warp have to arrive as one, and behind a branch that some of them took nothing else sees to that."""
    for kernel, body in kernels(name):
        for m in re.finditer(r"\bcluster_sync\(\);", body):
            assert re.search(r"__sync(warp|threads)\(\);\s*$", body[:m.start()]), (kernel, body[m.start() - 80:m.start()])
