"""Float32 blocks over the whole range of float32: features, weights and
gradients next to its largest value, against the formulas in 64 bits."""

import pytest
import torch

from mlx3d_amd.nn import gated_feed_forward
from test_gpu_feed_forward import formulas, outputs

pytestmark = pytest.mark.gpu

DEV = "cuda"
LARGEST = torch.finfo(torch.float32).max


# narrow in one operand and in several, narrow forward with a tiled backward, tiled
@pytest.mark.parametrize("widths", [(8, 24, 4), (40, 70, 20), (40, 70, 40), (200, 130, 70)],
                         ids=str)
@pytest.mark.parametrize("which", ("x", "w_gate", "w_down", "dy"))
@pytest.mark.parametrize("value", (LARGEST, -LARGEST, 3.395e38, 3.3895e38, 1e38))
def test_operands_next_to_the_largest(which, widths, value):
    """One operand holds the value in its last column, what it meets is small
    enough for every product and output to be finite."""
    d_in, hidden, d_out = widths
    g = torch.Generator().manual_seed(1)
    rows = 70

    def normal(*s):
        return torch.randn(s, generator=g)

    t = {"x": normal(rows, d_in), "w_gate": normal(hidden, d_in), "w_up": normal(hidden, d_in),
         "w_down": normal(d_out, hidden), "dy": normal(rows, d_out)}
    small = 2.0 ** -60
    if which == "x":
        t["x"][:, -1] = value
        t["w_gate"][:, -1] *= 2.0 ** -100
        t["w_up"][:, -1] *= 2.0 ** -100
        t["dy"] *= small
    elif which == "w_gate":
        t["w_gate"][-1] = value  # that channel's gate is far out on either side
        t["x"] *= 2.0 ** -100
        t["w_up"] /= small
    elif which == "w_down":
        t["w_down"][:, -1] = value
        t["w_up"] *= small
        t["dy"] *= small
    else:
        t["dy"][:, -1] = value
        t["w_down"] *= small
        t["w_up"] *= small
        t["x"] *= 2.0 ** -30
    args = [v.to(DEV) for v in t.values()]
    val, err = formulas(*args, "sigmoid")
    got = outputs(*args, "sigmoid")
    for name, v in val.items():
        # 2^-110: what products below the smallest normal number lose
        over = (got[name].double() - v).abs() - (1.02 * err[name] + 2.0 ** -23 * v.abs()
                                                 + 2.0 ** -110)
        held = v.abs() < 0.99 * LARGEST
        assert bool(held.any()) and bool((over[held] <= 0).all()), (name, float(over[held].max()))


@pytest.mark.parametrize("widths", [(8, 24, 4), (40, 70, 20), (200, 130, 70)], ids=str)
@pytest.mark.parametrize("size", (2.0 ** -100, 2.0 ** -112, 2.0 ** -120, 2.0 ** -130))
def test_small_operands_beside_the_largest(widths, size):
    """Weights far down meet features far up.  The narrow kernels hold a float32
    operand in three bfloat16 pieces, whose smallest is 2^-133; where products
    take subnormal pieces for 0, what is lost of an operand is below 2^-126."""
    d_in, hidden, d_out = widths
    g = torch.Generator().manual_seed(2)
    x = torch.randn((70, d_in), generator=g) * 2.0 ** 100
    wg, wu = torch.randn((2, hidden, d_in), generator=g) * size
    wd = torch.randn((d_out, hidden), generator=g)
    t = [v.to(DEV) for v in (x, wg, wu, wd)]
    y = gated_feed_forward(*t, activation="sigmoid")
    x, wg, wu, wd = (v.double() for v in t)
    g, u = x @ wg.T, x @ wu.T
    a = torch.sigmoid(g)
    lost = 2.0 ** -126 * x.abs().sum(dim=1, keepdim=True)
    eg = (d_in + 2) * 2.0 ** -24 * (x.abs() @ wg.abs().T) + lost
    eu = (d_in + 2) * 2.0 ** -24 * (x.abs() @ wu.abs().T) + lost
    h = a * u
    eh = (0.25 * eg + 2.0 ** -21 * (1 + g.abs())) * u.abs() + a * eu
    want = h @ wd.T
    err = eh @ wd.abs().T + (hidden + 2) * 2.0 ** -24 * (h.abs() @ wd.abs().T)
    over = (y.double() - want).abs() - (1.02 * err + 2.0 ** -110)
    assert bool((over <= 0).all()), float(over.max())
