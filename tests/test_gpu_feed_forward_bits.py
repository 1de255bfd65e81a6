"""The block's outputs carry the bits of their type: hidden channels and their
gradients reach the second products with more bits than 16-bit tensors hold,
and in float32's range, so that only the outputs are rounded."""

import pytest
import torch

from mlx3d_amd.nn import gated_feed_forward
from test_gpu_feed_forward import ROUND, act64, formulas, inputs, outputs

pytestmark = pytest.mark.gpu

DEV = "cuda"
HALVES = (torch.bfloat16, torch.float16)
# narrow widths with one operand a row and with several, streamed weights, tiled ones
SIZES = [(3000, 32, 128, 64), (1501, 27, 100, 21), (700, 60, 200, 50), (900, 128, 96, 120),
         (1100, 20, 300, 40), (33001, 128, 513, 250), (700, 200, 300, 130), (600, 512, 520, 512)]


def bounds(x, wg, wu, wd, dy, act):
    """Values in float64, and the bound of float32 arithmetic on these inputs
    whose hidden channels and gradients are held to 2^-16: two pieces of eight
    bits, in float16 also the product of second pieces that is left out (each
    2^-16 of a term at the very most, of either sign)."""
    val, err = formulas(*(t.float() for t in (x, wg, wu, wd, dy)), act)
    x, wg, wu, wd, dy = (t.double() for t in (x, wg, wu, wd, dy))
    g, u = x @ wg.T, x @ wu.T
    a, s = act64(g, act)
    dh = dy @ wd
    h, du, dg = a * u, dh * a, dh * u * s
    held = 2.0 ** -16
    err["y"] += held * (h.abs() @ wd.abs().T)
    err["dx"] += held * (dg.abs() @ wg.abs() + du.abs() @ wu.abs())
    err["dw_gate"] += held * (dg.abs().T @ x.abs())
    err["dw_up"] += held * (du.abs().T @ x.abs())
    err["dw_down"] += held * (dy.abs().T @ h.abs())
    return val, err


def check(got, val, err, dtype, names=None):
    r, sub = ROUND[dtype]
    for name in names or val:
        d = (got[name].double() - val[name]).abs()
        over = d - (1.02 * err[name] + r * val[name].abs() + sub)
        assert bool((over <= 0).all()), (name, float(over.max()), float(d.max()))


@pytest.mark.parametrize("dtype", HALVES, ids=str)
@pytest.mark.parametrize("act", ("silu", "gelu", "sigmoid"))
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_one_rounding(size, act, dtype):
    """One rounding to nearest leaves 0.38 to 0.41 of ROUND in the mean (a step's
    twelfth, over values spread through a power of two); a second one of the same
    size on the way 1.4 times as much."""
    t = inputs(*size, dtype, seed=sum(size))
    val, err = bounds(*t, act)
    got = outputs(*t, act)
    check(got, val, err, dtype)
    for name, v in val.items():
        rel = float((got[name].double() - v).norm() / v.norm())
        assert rel <= 0.47 * ROUND[dtype][0], (name, rel / ROUND[dtype][0])


# the last three channels of each hold the values, the others nothing
WIDTHS = [(8, 24, 4), (40, 70, 40), (128, 40, 6), (200, 130, 70)]


@pytest.mark.parametrize("dtype", HALVES, ids=str)
@pytest.mark.parametrize("widths", WIDTHS, ids=str)
def test_hidden_values_beyond_float16(widths, dtype):
    """h = 300 * 300 and 2000 * 2000, above what float16 holds, come down again
    with the weights; gradients of 2^-30 come up again."""
    d_in, hidden, d_out = widths
    rows = 70
    wg, wu = torch.zeros((2, hidden, d_in))
    wd = torch.zeros((d_out, hidden))
    wg[-1, -1] = wu[-1, -1] = 1.0
    wg[-2, -2] = wu[-2, -2] = 1.0
    wd[-1, -1] = 2.0 ** -4
    wd[-2, -2] = 2.0 ** -10
    x = torch.zeros((rows, d_in))
    x[:, -1] = 300.0 + torch.arange(rows)
    x[:, -2] = 2000.0 - 3 * torch.arange(rows)
    t = [v.to(dtype).to(DEV) for v in (x, wg, wu, wd, torch.zeros((rows, d_out)))]
    val, err = bounds(*t, "silu")
    check({"y": gated_feed_forward(*t[:4])}, val, err, dtype, ["y"])
    # the weight gradient sums h itself: dy = 2^-14
    t[4] = torch.full((rows, d_out), 2.0 ** -14).to(dtype).to(DEV)
    val, err = bounds(*t, "silu")
    check(outputs(*t, "silu"), val, err, dtype, ["y", "dw_down"])
    # small: dy = 2^-14, wd = 2^-16 (a float16 of one bit), wg = wu = 2^8
    wg[-1, -1] = wu[-1, -1] = 256.0
    wd[-1, -1] = 2.0 ** -16
    x[:, -1] = 0.004 + 1e-4 * torch.arange(rows)
    x[:, -2] = 0.0
    dy = torch.zeros((rows, d_out))
    dy[:, -1] = 2.0 ** -14
    t = [v.to(dtype).to(DEV) for v in (x, wg, wu, wd, dy)]
    val, err = bounds(*t, "silu")
    check(outputs(*t, "silu"), val, err, dtype)
