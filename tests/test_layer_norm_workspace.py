"""The workspace of the layer norm's gradient holds what the kernels use, and no more (no GPU
needed)."""

import pytest

from mlx3d_amd import _lib


@pytest.mark.parametrize("dtype", (0, 1, 2))
# rows of the widest teams, on both sides of what a workgroup holds, and the longest
@pytest.mark.parametrize("width, parts", ((1537, 512), (8192, 512), (8193, 256), (1 << 20, 256)))
@pytest.mark.parametrize("rows", (1, 255, 256, 257, 1024, 100_000))
def test_wide_rows_take_what_they_use(rows, width, parts, dtype):
    need = _lib.load().gsx_layer_norm_bwd_workspace_bytes(dtype, rows, width)
    used = min(rows, parts) * 2 * width * 4 + (rows * 12 if width > 8192 else 0)
    assert used <= need <= used + 512


@pytest.mark.parametrize("dtype", (0, 1, 2))
def test_no_width_takes_more_than_its_groups(dtype):
    L = _lib.load()
    for width in (1, 2, 3, 5, 7, 8, 9, 17, 32, 33, 64, 100, 127, 256, 513, 768, 1000, 1536):
        most = 1024 * 2 * width * 4
        last = 0
        for rows in (1, 2, 63, 1024, 1 << 18, 1 << 30):
            need = L.gsx_layer_norm_bwd_workspace_bytes(dtype, rows, width)
            assert 2 * width * 4 <= need <= min(most, rows * 2 * width * 4) + 512
            assert need >= last  # grows with the rows
            last = need
