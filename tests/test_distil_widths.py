"""A vocabulary that 32 bits do not hold is refused before anything is read or copied (no
GPU needed: the tensors have a shape and no data)."""

import pytest
import torch

from mlx3d_amd import _lib
from mlx3d_amd.losses import distillation_loss, distillation_value_and_grad


@pytest.mark.parametrize("call", (distillation_loss, distillation_value_and_grad))
@pytest.mark.parametrize("rows", (0, 4))
# 2^32 and a little more look like 0 and a small width to what keeps 32 bits of them
@pytest.mark.parametrize("vocab", (1 << 31, (1 << 32) - 1, 1 << 32, (1 << 32) + 9, (1 << 33) + 5))
def test_a_wide_vocabulary_is_refused(vocab, rows, call):
    logits = torch.empty((rows, vocab), dtype=torch.bfloat16, device="meta")
    values = torch.empty((rows, 2), device="meta")
    indices = torch.empty((rows, 2), dtype=torch.int64, device="meta")
    with pytest.raises(_lib.GsxError, match=r"gsx_distil_\w+ failed: .*\(status -4\)"):
        call(logits, values, indices)
