"""NaN logits beside the entries reach the loss of their row."""

import math

import pytest
import torch

from mlx3d_amd.losses import distillation_loss, distillation_value_and_grad

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16, torch.float16), ids=str)
@pytest.mark.parametrize("vocab", (3, 40, 9001))
@pytest.mark.parametrize("fill", (math.nan, -math.inf))
def test_nothing_but_nan_outside_the_entries(vocab, dtype, fill):
    """A row whose unnamed columns are all NaN, or one NaN among -inf."""
    g = torch.Generator().manual_seed(vocab)
    logits = torch.randn((5, vocab), generator=g)
    index = torch.stack([torch.randperm(vocab, generator=g)[:2] for _ in range(5)])
    values = torch.log(torch.tensor([[0.5, 0.3]])).expand(5, 2).contiguous()
    named = torch.zeros((5, vocab), dtype=torch.bool).scatter_(1, index, True)
    first = (~named).int().argmax(dim=1)
    for row in (1, 4):
        logits[row, ~named[row]] = fill
        logits[row, first[row]] = math.nan
    args = logits.to(dtype).to(DEV), values.to(DEV), index.to(DEV)
    each = distillation_loss(*args, teacher="log_probs", reduction="none")
    total, grad = distillation_value_and_grad(*args, teacher="log_probs", reduction="sum")
    assert each.isnan().tolist() == [False, True, False, False, True]
    assert math.isnan(float(total))
    assert grad.isnan().any(dim=1).tolist() == [False, True, False, False, True]
