"""The feature field's operators inside torch's checkpointing, whose saved
tensors may be read once: gradients as without it, with and without a graph of the
backward pass."""

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from mlx3d_amd.losses import distillation_loss
from mlx3d_amd.nn import gated_feed_forward

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.mark.parametrize("create_graph", (False, True))
@pytest.mark.parametrize("reentrant", (False, True))
def test_gradients_through_a_checkpoint(create_graph, reentrant):
    if create_graph and reentrant:
        pytest.skip("torch offers no graph of a reentrant checkpoint's backward")
    g = torch.Generator().manual_seed(0)
    x, wg, wu, wd = (torch.randn(s, generator=g).to(DEV).requires_grad_(True)
                     for s in ((50, 8), (16, 8), (16, 8), (9, 16)))
    index = torch.randint(0, 9, (50, 2), generator=g).to(DEV)
    values = torch.randn((50, 2), generator=g).to(DEV)

    def work(x, wg, wu, wd):
        return distillation_loss(gated_feed_forward(x, wg, wu, wd), values, index)

    leaves = (x, wg, wu, wd)
    want = torch.autograd.grad(work(*leaves), leaves)
    loss = checkpoint(work, *leaves, use_reentrant=reentrant)
    if reentrant:
        loss.backward()
        got = [v.grad for v in leaves]
    else:
        got = torch.autograd.grad(loss, leaves, create_graph=create_graph)
    for a, b in zip(got, want):
        assert torch.equal(a.detach(), b)
