"""GELU far out on the negative side, in 16 bits."""

import math

import pytest
import torch

from mlx3d_amd.nn import gated_feed_forward
from test_gpu_feed_forward import ROUND

pytestmark = pytest.mark.gpu

DEV = "cuda"
HALVES = (torch.bfloat16, torch.float16)
WIDTHS = [(8, 24, 4), (40, 70, 40), (128, 40, 6), (200, 130, 70)]


@pytest.mark.parametrize("dtype", HALVES, ids=str)
@pytest.mark.parametrize("widths", WIDTHS, ids=str)
def test_the_tail_of_gelu(widths, dtype):
    """g Phi(g) far out on the negative side, to the relative precision of the
    type: 2^14 and 2^12 bring what is left there back into float16's range."""
    d_in, hidden, d_out = widths
    gate = torch.linspace(-5.5, -2.0, 90)
    x = torch.zeros((90, d_in))
    x[:, -1], x[:, -2] = gate, 2.0 ** 14
    wg, wu = torch.zeros((2, hidden, d_in))
    wg[-1, -1] = wu[-1, -2] = 1.0
    wd = torch.zeros((d_out, hidden))
    wd[-1, -1] = 2.0 ** 2
    t = [v.to(dtype).to(DEV) for v in (x, wg, wu, wd)]
    y = gated_feed_forward(*t, activation="gelu")[:, -1].double().cpu()
    g = t[0][:, -1].double().cpu()
    want = 2.0 ** 16 * g * 0.5 * torch.special.erfc(-g / math.sqrt(2))
    r, sub = ROUND[dtype]
    assert bool(((y - want).abs() <= (r + 2.0 ** -14) * want.abs() + sub).all()), \
        float(((y - want) / want).abs().max())
