"""Float32 exponents of the distillation loss to a unit of the power, however
far a logit lies below its row's maximum."""

import pytest
import torch

from mlx3d_amd.losses import distillation_value_and_grad

pytestmark = pytest.mark.gpu

DEV = "cuda"
U32 = 2.0 ** -24


@pytest.mark.parametrize("temp", (1.0, 1.5, 3.933349609375, 2.790283203125, 0.485107421875))
@pytest.mark.parametrize("vocab", (64, 300, 2000, 6000))
def test_ratios_of_gradients(vocab, temp):
    """Whole logits, whose differences are exact: gradients outside the entry
    stand to each other as exp(difference / T) to the powers' rounding (three U32
    each), the factors' (one each) and 2^-6 of one for a unit of the exponent."""
    logits = -(torch.arange(vocab) % 64).float().expand(3, vocab).contiguous()
    index = torch.zeros((3, 1), dtype=torch.int64)
    _, g = distillation_value_and_grad(logits.to(DEV), torch.zeros((3, 1), device=DEV),
                                       index.to(DEV), temperature=temp, reduction="sum")
    z = (logits.double() / temp)[:, 1:]
    g = g.double().cpu()[:, 1:]
    off = torch.where(z > -80, ((g / g[:, :1]).log() - (z - z[:, :1])).abs(), 0)
    assert bool((off <= U32 * (9 + z.abs() / 32)).all()), float(off.max()) / U32


@pytest.mark.parametrize("vocab", (150, 2048, 50_000))
@pytest.mark.parametrize("teacher", ("logits", "log_probs"))
def test_no_further_off_than_elementary_operations(vocab, teacher):
    """Against 64 bits, in the mean: the differences' rounding, which elementary
    float32 operations have as well, and not the exponents'."""
    g = torch.Generator().manual_seed(vocab)
    logits = torch.randn((64, vocab), generator=g).mul_(4).to(DEV)
    values, index = torch.randn((64, 9), generator=g).topk(9, dim=1)
    if teacher == "log_probs":
        values = torch.log_softmax(values, 1) - 0.5
    values, index = values.to(DEV), index.to(DEV)
    _, grad = distillation_value_and_grad(logits, values, index, teacher=teacher, reduction="sum")

    def rest(z):  # the gradient outside the entries, up to a factor of the row
        p = torch.exp(z - z.amax(dim=1, keepdim=True))
        return p / p[:, 20:21]

    want = rest(logits.double())[:, 20:]
    own = (grad / grad[:, 20:21])[:, 20:].double()
    plain = rest(logits)[:, 20:].double()
    off = [float(((v - want) / want).square().mean().sqrt()) for v in (own, plain)]
    assert off[0] <= 1.25 * off[1], off
