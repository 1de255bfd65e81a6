"""What float32 rounding may do to the distillation loss's exponents, logarithms
and quotients, one at a time, on rows whose sums are exact."""

import math

import pytest
import torch

from mlx3d_amd.losses import distillation_loss, distillation_value_and_grad

pytestmark = pytest.mark.gpu

DEV = "cuda"
U32 = 2.0 ** -24


# temperatures at which log2(e) / T rounds by less than half of U32, and by 1.8 where
# log2(e) and 1 / T are rounded before their product is
@pytest.mark.parametrize("temp", (3.933349609375, 2.790283203125, 0.485107421875))
@pytest.mark.parametrize("vocab", (64, 2000, 6000))
def test_exponents(vocab, temp):
    """Whole logits: gradients outside the entry stand to each other as
    exp(difference / T), to the rounding of log2(e) / T (half a U32 of the exponent)
    and of the product (one), of the powers (two each) and the factors (one each)."""
    logits = -(torch.arange(vocab) % 64).float().expand(3, vocab).contiguous()
    index = torch.zeros((3, 1), dtype=torch.int64)
    _, g = distillation_value_and_grad(logits.to(DEV), torch.zeros((3, 1), device=DEV),
                                       index.to(DEV), temperature=temp, reduction="sum")
    z = logits.double() / temp
    got = (g.double().cpu()[:, 1:] / g.double().cpu()[:, 1:2]).log()
    off = torch.where(z[:, 1:] > -80, (got - (z[:, 1:] - z[:, 1:2])).abs(), 0)  # normal numbers
    assert bool((off <= U32 * (1.52 * (z[:, 1:] + z[:, 1:2]).abs() + 8)).all()), \
        float((off / (U32 * z[:, 1:].abs().clamp(min=1))).max())


@pytest.mark.parametrize("teacher", ("logits", "log_probs"))
def test_logarithms_and_quotients(teacher):
    """Equal logits, whose sum is V itself: the loss is its float32 logarithm, bit
    for bit, and each gradient 1 / V, to its own rounding."""
    for vocab in (*range(2, 130), 255, 1000, 1023, 2047, 3001, 4099, 10007):
        logits = torch.zeros((2, vocab), device=DEV)
        args = logits, torch.zeros((2, 1), device=DEV), torch.zeros((2, 1), dtype=torch.int64,
                                                                   device=DEV)
        each = distillation_loss(*args, teacher=teacher, reduction="none")
        want = torch.full((2,), float(vocab), device=DEV).log()
        assert torch.equal(each, want), (vocab, float(each[0]), math.log(vocab))
        _, g = distillation_value_and_grad(*args, teacher=teacher, reduction="sum")
        off = (g[:, 1:].double() * vocab - 1).abs()
        assert bool((off <= 1.01 * U32).all()), (vocab, float(off.max()) / U32)
