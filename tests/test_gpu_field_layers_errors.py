"""What goes wrong in a gradient of the field layers reaches the caller as what it is: a
``GsxError``, as from a forward call.  The saved tensors are replaced by larger ones than the
entry points take, which refuse them before any launch."""

import threading

import pytest
import torch

from mlx3d_amd import _lib
from mlx3d_amd.nn import embedding, layer_norm

pytestmark = pytest.mark.gpu

DEV = "cuda"


def norm():
    """A norm whose saved rows come back wider than 2^20 columns."""
    leaf = torch.ones((1, 4), device=DEV, requires_grad=True)
    with torch.autograd.graph.saved_tensors_hooks(
            lambda t: t, lambda t: torch.zeros((1, (1 << 20) + 1), device=DEV)):
        weight = torch.ones((4,), device=DEV, requires_grad=True)
        return layer_norm(leaf, None, weight), [leaf, weight]


def lookup():
    """A lookup whose saved indices come back as more than 2^30 (never read)."""
    leaf = torch.ones((3, 1), device=DEV, requires_grad=True)
    with torch.autograd.graph.saved_tensors_hooks(
            lambda t: t,
            lambda t: torch.empty(((1 << 30) + 1,), dtype=torch.int32, device=DEV)):
        return embedding(torch.zeros((2,), dtype=torch.int32, device=DEV), leaf), [leaf]


CASES = ((norm, "gsx_layer_norm_bwd_workspace_bytes"), (lookup, "gsx_embed_bwd_workspace_bytes"))


def still_right():
    x = torch.randn((5, 6), device=DEV, requires_grad=True)
    (g,) = torch.autograd.grad(layer_norm(x).sum(), x)
    assert g.shape == x.shape and bool(g.isfinite().all())


@pytest.mark.parametrize("create_graph", (False, True))
@pytest.mark.parametrize("make, entry", CASES, ids=("norm", "lookup"))
def test_a_failing_gradient_raises_a_gsx_error(make, entry, create_graph):
    for _ in range(2):
        y, leaves = make()
        with pytest.raises(_lib.GsxError, match=entry + r" failed: .*\(status -4\)"):
            torch.autograd.grad(y, leaves, torch.ones_like(y), create_graph=create_graph)
    still_right()


@pytest.mark.parametrize("make, entry", CASES, ids=("norm", "lookup"))
def test_from_another_thread(make, entry):
    y, _ = make()
    caught = []

    def run():
        try:
            y.backward(torch.ones_like(y))
        except Exception as e:
            caught.append(e)

    t = threading.Thread(target=run)
    t.start()
    t.join()
    assert len(caught) == 1 and type(caught[0]) is _lib.GsxError and entry in str(caught[0])
    still_right()


def test_other_errors_keep_their_type():
    """A second derivative is refused as before."""
    x = torch.randn((5, 6), device=DEV, requires_grad=True)
    (g,) = torch.autograd.grad(layer_norm(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable") as e:
        g.sum().backward()
    assert not isinstance(e.value, _lib.GsxError)
