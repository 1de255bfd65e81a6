"""Rows in several stretches, whose weight gradients add up: against the
formulas, and each row's results as they are among fewer rows."""

import pytest
import torch

from test_gpu_feed_forward import TYPES, check, formulas, inputs, outputs

pytestmark = pytest.mark.gpu


# more than 1 GB of hidden channels (tiled) or of the groups' parts of dx (narrow),
# the last stretch shorter; one split of the weights' gradients and several
SIZES = [(300_001, 130, 2000, 10), (300_017, 3, 2000, 130), (90_011, 200, 6000, 40),
         (900_007, 120, 600, 8)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_several_stretches(size, dtype):
    x, wg, wu, wd, dy = inputs(*size, dtype, seed=size[0])
    got = outputs(x, wg, wu, wd, dy, "silu")
    rows = size[0]
    total, bound = {}, {}
    for at in range(0, rows, 50_000):  # doubles of all rows at once would take 20 GB
        part = slice(at, at + 50_000)
        val, err = formulas(x[part], wg, wu, wd, dy[part], "silu")
        check({k: got[k][part] for k in ("y", "dx")}, {k: val[k] for k in ("y", "dx")}, err, dtype)
        for k in ("dw_gate", "dw_up", "dw_down"):
            total[k] = total.get(k, 0) + val[k]
            bound[k] = bound.get(k, 0) + err[k]
    if dtype == torch.float32:  # one sum of all rows instead of 50 000
        for k in bound:
            bound[k] = bound[k] * (rows / 50_000 + 1)
    check({k: got[k] for k in total}, total, bound, dtype)


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16), ids=str)
def test_a_row_does_not_depend_on_its_stretch(dtype):
    x, wg, wu, wd, dy = inputs(200_003, 130, 2000, 10, dtype, seed=1)
    whole = outputs(x, wg, wu, wd, dy, "silu")
    for first, n in ((0, 700), (99_900, 400), (100_100, 300), (200_000, 3)):
        part = outputs(x[first:first + n], wg, wu, wd, dy[first:first + n], "silu")
        for k in ("y", "dx"):
            assert torch.equal(part[k], whole[k][first:first + n]), (k, first)
    again = outputs(x, wg, wu, wd, dy, "silu")
    assert all(torch.equal(whole[k], again[k]) for k in whole)
