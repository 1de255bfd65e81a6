"""The short rows' kernels at both ends of every choice of lanes, words and
entries a lane, in each type and for both teachers."""

import pytest
import torch

from mlx3d_amd.losses import distillation_loss, distillation_value_and_grad
from test_gpu_distil import TEACHERS, TYPES, definition, inputs, near_rows

pytestmark = pytest.mark.gpu


def words(dtype, vocab):
    return vocab if dtype == torch.float32 else (vocab + 1) // 2 + 1


def lanes(dtype, vocab, top):
    g = 4
    while g < 64 and (g * 14 < words(dtype, vocab) or g * 4 < top):
        g *= 2
    return g


def sizes(dtype):
    """(vocab, top) on both sides of each number of words a lane, for one, two
    and four entries a lane, as far as rows of 8 KB go."""
    size = 4 if dtype == torch.float32 else 2
    found = set()
    for g in (4, 8, 16, 32, 64):
        for n in (3, 6, 8, 10, 14, 20, 33):
            for vocab in ((n * g, n * g + 1) if size == 4 else (2 * n * g - 3, 2 * n * g - 1)):
                vocab = min(vocab, 8192 // size)
                for top in (3, 2 * g - 1, 4 * g - 1, 4 * g):
                    if 1 <= top <= min(vocab, 256) and lanes(dtype, vocab, top) == g:
                        found.add((vocab, top))
    return sorted(found)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("teacher", TEACHERS)
def test_every_choice(dtype, teacher):
    for vocab, top in sizes(dtype):
        rows = 5 if vocab > 600 else 19
        logits, values, index = inputs(rows, vocab, top, dtype, teacher, seed=vocab + top)
        loss, grad, loss_tol, grad_tol, _ = definition(logits, values, index, 1.5, teacher)
        how = dict(temperature=1.5, teacher=teacher)
        total, g = distillation_value_and_grad(logits, values, index, reduction="sum", **how)
        near_rows(total, loss.sum(), loss_tol.sum())
        near_rows(g, grad, grad_tol, dtype)
        each = distillation_loss(logits, values, index, reduction="none", **how)
        near_rows(each, loss, loss_tol)
