"""Widths of the decoder that 32 bits do not hold are refused before anything is read or
copied (no GPU needed: the tensors have a shape and no data)."""

import pytest
import torch

from mlx3d_amd import _lib
from mlx3d_amd.nn import gated_feed_forward

# 2^32 and a little more look like 0 and a small width to what keeps 32 bits of them
WIDTHS = (1 << 31, (1 << 32) - 1, 1 << 32, (1 << 32) + 8, (1 << 33) + 1)


def shaped(*shape):
    return torch.empty(shape, dtype=torch.bfloat16, device="meta")


@pytest.mark.parametrize("which", ("d_in", "hidden", "d_out"))
@pytest.mark.parametrize("width", WIDTHS)
def test_a_wide_block_is_refused(width, which):
    size = {"d_in": 8, "hidden": 16, "d_out": 3, which: width}
    gate, up = (shaped(size["hidden"], size["d_in"]) for _ in range(2))
    for rows in (0, 4):
        with pytest.raises(_lib.GsxError, match=r"gsx_ffn_fwd failed: .*\(status -4\)"):
            gated_feed_forward(shaped(rows, size["d_in"]), gate, up,
                               shaped(size["d_out"], size["hidden"]))
