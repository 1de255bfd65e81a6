"""Temperatures whose reciprocal float32 cannot hold are refused by both
layers, before any launch (no GPU needed)."""

import ctypes

import pytest
import torch

from mlx3d_amd import _lib
from mlx3d_amd.losses import distillation_loss

P = ctypes.c_void_p(4096)  # never dereferenced


def call(temp):
    return distillation_loss(torch.zeros((4, 9)), torch.zeros((4, 2)),
                             torch.zeros((4, 2), dtype=torch.int64), temperature=temp)


@pytest.mark.parametrize("temp", (1e-50, 1e-40, 2.0 ** -149, 9e-39, -1e-20))
def test_too_small(temp):
    with pytest.raises(ValueError, match="temperature"):
        call(temp)
    assert _lib.load().gsx_distil_fwd(0, 4, 9, 2, P, 9, P, P, 0, temp, 0, 2, P, P, 1 << 40,
                                      None) == -1


@pytest.mark.parametrize("temp", (1e-37, 2.0 ** -126, 1.0, 1e37))
def test_accepted(temp):
    with pytest.raises(ValueError, match="GPU only"):  # the next check
        call(temp)
    assert _lib.load().gsx_distil_fwd(0, 4, 9, 2, P, 9, P, P, 0, temp, 0, 2, P, P, 16,
                                      None) == -3  # the next one
