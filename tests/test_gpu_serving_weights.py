"""Attention over pages of e4m3 whose value vectors are zeros, or far smaller than others, under keys that have much of the weight: what a cell adds to the
sum of a row's weights has nothing to do with the size of its value.  The comparison and its tolerances are those of ``test_gpu_serving_ops.py``: they count
in parts of sum p |v| / sum p, so a weight that is lost shows as soon as it is 2^-8 of its row's sum.

A probability's product with a value of 2^-k of the row's largest is of a float16 number 2^k smaller: it is right to 2^-11 of itself down to 2^-21 of the
largest and to 2^-32 of the largest below that, which 2,000 cells make 2^-21 of sum p |v| where entries of the larger values are not zeros."""
import pytest
import torch

from tests.test_gpu_serving_ops import Problem

pytestmark = pytest.mark.gpu

# one row a KV head, several, many; head sizes of both kernels
SHAPES = [(4, 4, 128, [1, 1, 1]), (16, 2, 128, [1, 2, 1]), (32, 2, 64, [1, 1, 1]), (12, 2, 96, [1, 64, 9]), (8, 2, 32, [5, 33, 1]), (32, 8, 128, [64, 1, 30]), (8, 2, 64, [20, 64, 3])]


def problem(shape, sharp, seed=0):
    H, G, D, lens = shape
    return Problem(lens, [300, 70, 1100], H, G, D, True, tree=True, seed=seed, sharp=sharp)


def shrink(p, cells, by):
    """The values of these cells (a slice of every page's) smaller by 2^by, or zeros: as ``rope_kv_store`` writes them."""
    if by is None:
        p.v.view(torch.uint8)[:, :, cells] = 0
        p.ve[:, :, cells] = 67
    else:
        p.ve[:, :, cells] = (p.ve[:, :, cells].int() - by).clamp(67, 246).to(torch.uint8)


@pytest.mark.parametrize("by", [None, 16, 24, 40])
@pytest.mark.parametrize("sharp", [0.0, 0.3])
@pytest.mark.parametrize("shape", SHAPES)
def test_weights_of_small_values_count(shape, sharp, by):
    """Half of the cells, and all but a few; with equal scores too."""
    for cells in (slice(1, None, 2), slice(3, None)):
        p = problem(shape, sharp)
        shrink(p, cells, by)
        for n_splits in (None, 1, 3, 12):
            p.check(p.run(n_splits=n_splits))


@pytest.mark.parametrize("shape", SHAPES)
def test_a_cell_of_zeros_that_has_most_of_the_weight(shape):
    """The first cell's value is zeros and its key is near to every query, as an attention sink's."""
    H, G, D, lens = shape
    p = problem(shape, 0.2, seed=1)
    p.q += 1.0
    for row in p.table:
        p.v.view(torch.uint8)[row[0], :, 0] = 0
        p.ve[row[0], :, 0] = 67
        p.k.view(torch.uint8)[row[0], :, 0] = 0x38         # 1.0
        p.ke[row[0], :, 0] = 127
    for n_splits in (None, 1, 5, 12):
        p.check(p.run(n_splits=n_splits))


@pytest.mark.parametrize("whole_pages", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_weights_beside_values_near_the_end_of_the_range(shape, whole_pages):
    """Values of about 2^100, beside zeros and beside values 2^60 and 2^140 smaller: in the same page, and in pages of their own."""
    for by in (None, 60, 140):
        p = problem(shape, 0.3, seed=2)
        p.ve.copy_((p.ve.int() + 100).clamp(67, 246).to(torch.uint8))
        if whole_pages:
            for row in p.table:
                for page in row[1::2] if len(row) > 3 else row[:1]:
                    if page >= 0:
                        if by is None:
                            p.v.view(torch.uint8)[page] = 0
                        p.ve[page] = 67 if by is None else (p.ve[page].int() - by).clamp(67, 246).to(torch.uint8)
        else:
            shrink(p, slice(1, None, 2), by)
        for n_splits in (1, 3, 12):
            p.check(p.run(n_splits=n_splits))
