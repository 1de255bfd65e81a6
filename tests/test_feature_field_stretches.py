"""Workspaces of many rows are bounded, and shapes whose hidden channels take
more workgroups than one launch holds are accepted (no GPU needed)."""

import pytest

from mlx3d_amd import _lib

GB = 1 << 30


# dtype, act, rows, d_in, hidden, d_out
@pytest.mark.parametrize("head, forward, backward", [
    ((0, 0, 921_600, 64, 512, 64), 1, 4),          # a 720p view, tiled backward
    ((1, 0, 97_000_000, 200, 1365, 64), 1, 4),     # 2^24 workgroups of hidden channels
    ((1, 0, 1 << 30, 2, 70, 300), 1, 4),
    ((1, 0, 2_073_600, 128, 2048, 64), 0, 2),      # 16 groups of the narrow backward
    ((1, 0, 1 << 30, 1, 2048, 1), 0, 2),
])
def test_bounded(head, forward, backward):
    L = _lib.load()
    assert 0 <= L.gsx_ffn_fwd_workspace_bytes(*head) <= forward * GB
    assert 0 < L.gsx_ffn_bwd_workspace_bytes(*head) <= backward * GB


def test_one_stretch_holds_what_it_needs():
    """Few rows: arrays of the rows' own size."""
    L = _lib.load()
    assert L.gsx_ffn_fwd_workspace_bytes(0, 0, 1000, 200, 64, 8) == 1000 * 64 * 4
    assert L.gsx_ffn_bwd_workspace_bytes(0, 0, 100, 200, 64, 8) == 3 * 100 * 64 * 4


@pytest.mark.parametrize("head", [(2, 0, 921_600, 200, 512, 64), (2, 0, 97_000_000, 200, 1365, 64),
                                  (2, 0, 1 << 30, 2, 70, 300), (2, 0, 2_073_600, 512, 40, 128)])
def test_float16_pieces_are_bounded_too(head):
    """The rows' two pieces stand beside three hidden arrays, the weights' once."""
    L = _lib.load()
    weights = 4 * (head[4] + 8) * (2 * (head[3] + 8) + head[5] + 8)
    assert 0 <= L.gsx_ffn_fwd_workspace_bytes(*head) <= GB + weights
    sums = 512 * 8192 * 4 * 3 + 3 * weights
    assert 0 < L.gsx_ffn_bwd_workspace_bytes(*head) <= 5 * GB + weights + sums
