"""Workspaces that are too small or missing, for the shapes that write to one,
checked on the host before any launch (no GPU needed)."""

import ctypes

import pytest

from mlx3d_amd import _lib

SHORT = -3  # GSX_ERR_WORKSPACE
BUF = (ctypes.c_char * 4096)()
P = ctypes.c_void_p((ctypes.addressof(BUF) + 255) // 256 * 256)  # never dereferenced


# dtype, act, rows, d_in, hidden, d_out: tiled widths in each type, one row, many
@pytest.mark.parametrize("head", [(0, 0, 4, 200, 64, 8), (1, 1, 1, 129, 1, 1),
                                  (2, 2, 100_000, 512, 1365, 512), (0, 0, 30_000, 8, 4000, 300)])
def test_the_tiled_forward_refuses(head):
    L = _lib.load()
    need = L.gsx_ffn_fwd_workspace_bytes(*head)
    assert need > 0
    d_in = head[3]
    call = (*head, P, d_in, P, P, P, P)
    assert L.gsx_ffn_fwd(*call, P, need - 1, None) == SHORT
    assert L.gsx_ffn_fwd(*call, P, 0, None) == SHORT
    assert L.gsx_ffn_fwd(*call, None, need, None) == SHORT
    assert L.gsx_ffn_fwd(*call, ctypes.c_void_p(P.value + 8), need, None) == -1


@pytest.mark.parametrize("head", [(0, 0, 4, 8, 8, 8), (0, 0, 4, 200, 64, 8), (1, 1, 1, 129, 1, 1),
                                  (2, 2, 100_000, 512, 1365, 512), (1, 0, 5000, 32, 1000, 32)])
def test_the_backward_refuses(head):
    L = _lib.load()
    need = L.gsx_ffn_bwd_workspace_bytes(*head)
    assert need > 0
    d_in, d_out = head[3], head[5]
    call = (*head, P, d_in, P, P, P, P, d_out, P, P, P, P)
    assert L.gsx_ffn_bwd(*call, P, need - 1, None) == SHORT
    assert L.gsx_ffn_bwd(*call, None, need, None) == SHORT
    assert L.gsx_ffn_bwd(*call, ctypes.c_void_p(P.value + 8), need, None) == -1
