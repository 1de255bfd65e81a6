"""The feature field's operators have no second derivatives, and say so: a
penalty on their gradients raises an error and never loses its term."""

import pytest
import torch

from mlx3d_amd.losses import distillation_loss
from mlx3d_amd.nn import gated_feed_forward

pytestmark = pytest.mark.gpu

DEV = "cuda"


def block():
    g = torch.Generator().manual_seed(0)
    x, wg, wu, wd = (torch.randn(s, generator=g).to(DEV).requires_grad_(True)
                     for s in ((9, 8), (16, 8), (16, 8), (3, 16)))
    return gated_feed_forward(x, wg, wu, wd).sum(), x


def loss():
    g = torch.Generator().manual_seed(0)
    logits = torch.randn((9, 8), generator=g).to(DEV).requires_grad_(True)
    index = torch.zeros((9, 1), dtype=torch.int64, device=DEV)
    return distillation_loss(logits, torch.zeros((9, 1), device=DEV), index), logits


@pytest.mark.parametrize("make", (block, loss))
def test_a_penalty_on_the_gradient_is_refused(make):
    value, leaf = make()
    (grad,) = torch.autograd.grad(value, leaf, create_graph=True)
    objective = leaf.square().sum() + grad.square().sum()
    with pytest.raises(RuntimeError, match="once_differentiable"):
        objective.backward()


@pytest.mark.parametrize("make", (block, loss))
def test_first_derivatives_stay(make):
    value, leaf = make()
    (kept,) = torch.autograd.grad(value, leaf, create_graph=True)
    value, leaf = make()
    (plain,) = torch.autograd.grad(value, leaf)
    assert torch.equal(kept, plain)
