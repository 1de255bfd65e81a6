"""Sizes at the ends of what the embedding and the layer norm take, through their public
calls: what is too large is refused before any launch."""

import contextlib

import pytest
import torch

from mlx3d_amd import _lib
from mlx3d_amd.nn import embedding, layer_norm

pytestmark = pytest.mark.gpu

DEV = "cuda"
# from the limit to what 32 bits do not hold, and to what looks like a small width in them
WIDTHS = ((1 << 20) + 1, 1 << 31, 1 << 32, (1 << 32) + 64)


@contextlib.contextmanager
def refused(entry):
    """A ``GsxError`` before more than a copy of three rows of 2^20 + 1 is allocated (these
    are copied first, being one element repeated)."""
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    with pytest.raises(_lib.GsxError, match=entry + r" failed: .*\(status -4\)"):
        yield
    assert torch.cuda.max_memory_allocated() < before + (1 << 26)


@pytest.mark.parametrize("rows", (0, 1, 3))
@pytest.mark.parametrize("width", WIDTHS)
def test_a_norm_that_is_too_wide_is_refused(width, rows):
    x = torch.zeros((1, 1), dtype=torch.bfloat16, device=DEV).expand(rows or 1, width)[:rows]
    with refused("gsx_layer_norm_fwd"):
        layer_norm(x)


@pytest.mark.parametrize("count", (0, 3))
@pytest.mark.parametrize("width", WIDTHS)
def test_a_table_that_is_too_wide_is_refused(width, count):
    table = torch.zeros((1, 1), dtype=torch.bfloat16, device=DEV).expand(2, width)
    with refused("gsx_embed_fwd"):
        embedding(torch.zeros((count,), dtype=torch.int64, device=DEV), table)


def test_the_widest_rows_are_taken():
    width = 1 << 20
    x = torch.arange(width, device=DEV, dtype=torch.float32).expand(2, width)
    y = layer_norm(x)
    assert y.shape == x.shape and bool(y.isfinite().all())
    table = x.contiguous()
    assert torch.equal(embedding(torch.tensor([1], device=DEV), table), table[1:])
