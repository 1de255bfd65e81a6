"""Widths that 32 bits do not hold are refused by the field layers' nodes, before anything is
read, copied or launched (no GPU needed: the tensors have a shape and no data)."""

import pytest
import torch

from mlx3d_amd import _lib

# 2^32 and a little more look like 0 and a small width to what keeps 32 bits of them
WIDTHS = (1 << 31, (1 << 32) - 1, 1 << 32, (1 << 32) + 64, (1 << 33) + 1)


def shaped(rows, width, dtype=torch.bfloat16):
    return torch.empty((rows, width), dtype=dtype, device="meta")


@pytest.mark.parametrize("width", WIDTHS)
def test_a_wide_table_is_refused(width):
    for count in (0, 4):
        with pytest.raises(_lib.GsxError, match=r"gsx_embed_fwd failed: .*\(status -4\)"):
            _lib.autograd().embedding(torch.zeros((count,), dtype=torch.int64), shaped(3, width), 1.0)


@pytest.mark.parametrize("rows", (0, 1, 5))
@pytest.mark.parametrize("width", WIDTHS)
def test_a_wide_norm_is_refused(width, rows):
    weight = shaped(1, width)[0]
    for w, b in ((None, None), (weight, None), (weight, weight)):
        with pytest.raises(_lib.GsxError, match=r"gsx_layer_norm_fwd failed: .*\(status -4\)"):
            _lib.autograd().layer_norm(shaped(rows, width), w, b, 1e-5)


def test_a_wide_norm_without_rows_on_the_host():
    """Rows are counted by division; no row is needed for that to go wrong."""
    with pytest.raises(_lib.GsxError, match=r"\(status -4\)"):
        _lib.autograd().layer_norm(torch.empty((0, 1 << 32)), None, None, 1e-5)
