"""The narrow kernels' long walks: workgroups of the backward that take five
tiles of 32 rows and more (sums of the weight gradients carried along, both places
of the staged tile used again, the last tile ragged), one to four pairs of waves and
several groups of them; the forward's weights staged again for every 256 rows, and
its workgroups' second walk."""

import pytest
import torch

from mlx3d_amd.nn import gated_feed_forward
from test_gpu_feed_forward import TYPES, check, formulas, inputs, outputs

pytestmark = pytest.mark.gpu

# rows for five tiles or more of every workgroup in 16 bits, where there are most
# workgroups: 2048 / pairs of them for one group, 512 / groups for more
BACKWARD = [(330_013, 32, 20, 64), (164_005, 27, 40, 21), (110_003, 16, 70, 33),
            (82_017, 32, 128, 64), (28_001, 32, 300, 64), (164_001, 64, 33, 32),
            (82_003, 40, 128, 16), (82_001, 8, 100, 100), (20_009, 128, 600, 30),
            (20_011, 100, 130, 50), (82_011, 128, 90, 64)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("size", BACKWARD, ids=str)
def test_many_tiles_of_a_workgroup(size, dtype):
    t = inputs(*size, dtype, seed=size[0])
    check(outputs(*t, "silu"), *formulas(*t, "silu"), dtype)


# weights over 144 KB in float32 (16 bits for the third) on both sides of where they
# are streamed, the last stretch of chunks a partial one
FORWARD = [(20, 300, 40), (64, 700, 100), (128, 513, 256), (32, 1365, 64)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows", (32_767, 32_768, 33_001, 140_001))
@pytest.mark.parametrize("widths", FORWARD, ids=str)
def test_streamed_weights(widths, rows, dtype):
    x, wg, wu, wd, dy = inputs(rows, *widths, dtype, seed=3)
    y = gated_feed_forward(x, wg, wu, wd, activation="gelu")
    for part in (slice(0, 600), slice(rows // 2, rows // 2 + 600), slice(rows - 600, rows)):
        val, err = formulas(x[part], wg, wu, wd, dy[part], "gelu")
        check({"y": y[part]}, {"y": val["y"]}, err, dtype)


@pytest.mark.parametrize("rows", (65_537, 70_001, 131_073))
def test_second_walk_with_resident_weights(rows):
    t = inputs(rows, 32, 128, 64, torch.float32, seed=4)
    val, err = formulas(*t, "silu")
    check({"y": gated_feed_forward(*t[:4])}, {"y": val["y"]}, err, torch.float32)
