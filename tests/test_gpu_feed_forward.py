"""The gated feed-forward block against its formulas in 64 bits, gradients
against differences, and its layouts.

Each output is held to a running error bound: what float32 sums and the
roundings to the tensors' type can do, first order, from the magnitudes of the
terms (computed here in float64 beside the values)."""

import math

import pytest
import torch

from mlx3d_amd.nn import GatedFeedForward, gated_feed_forward

pytestmark = pytest.mark.gpu

DEV = "cuda"
U32 = 2.0 ** -24
# the unit roundoff of 8 and 11 significant bits, and half the smallest subnormal
ROUND = {torch.float32: (0.0, 0.0), torch.bfloat16: (2.0 ** -8, 2.0 ** -134),
         torch.float16: (2.0 ** -11, 2.0 ** -25)}
# largest |act'| and |act''|
LIPSCHITZ = {"silu": (1.1, 0.5), "gelu": (1.13, 0.8), "sigmoid": (0.25, 0.1)}
ACTS = ("silu", "gelu", "sigmoid")
TYPES = (torch.float32, torch.bfloat16, torch.float16)

# (rows, d_in, hidden, d_out): one row, ragged everywhere, tile edges on both
# sides, one of each width, wide and narrow
SIZES = [(1, 32, 64, 21), (1, 1, 1, 1), (2, 3, 5, 7), (63, 32, 128, 64), (64, 32, 32, 16),
         (65, 27, 100, 21), (129, 33, 65, 17), (257, 64, 96, 48), (130, 31, 33, 1),
         (1000, 16, 256, 128), (517, 128, 40, 3), (300, 200, 300, 130), (77, 5, 257, 65),
         (1500, 48, 130, 80), (40, 512, 520, 512), (4099, 32, 128, 64)]


def inputs(rows, d_in, hidden, d_out, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)

    def n(*s):
        return torch.randn(s, generator=g)

    x = n(rows, d_in) * 2.0
    wg, wu = n(hidden, d_in) / math.sqrt(d_in), n(hidden, d_in) / math.sqrt(d_in)
    wd = n(d_out, hidden) / math.sqrt(hidden)
    dy = n(rows, d_out)
    return [t.to(dtype).to(DEV) for t in (x, wg, wu, wd, dy)]


def act64(g, act):
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(g / math.sqrt(2)))
        return g * cdf, cdf + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(g)
    return (s, s * (1 - s)) if act == "sigmoid" else (g * s, s * (1 + g * (1 - s)))


def formulas(x, wg, wu, wd, dy, act):
    """Values in float64 and a bound of each output's error."""
    dtype = x.dtype
    r, sub = ROUND[dtype]
    x, wg, wu, wd, dy = (t.double() for t in (x, wg, wu, wd, dy))
    rows, d_in = x.shape
    hidden, d_out = wd.shape[1], wd.shape[0]
    l1, l2 = LIPSCHITZ[act]
    g, u = x @ wg.T, x @ wu.T
    eg = (d_in + 2) * U32 * (x.abs() @ wg.abs().T)
    eu = (d_in + 2) * U32 * (x.abs() @ wu.abs().T)
    a, s = act64(g, act)
    ea = l1 * eg + 8 * U32 * (a.abs() + g.abs())
    es = l2 * eg + 16 * U32 * (1 + g.abs())
    h = a * u

    def rounded(v):
        return r * v.abs() + sub

    eh = ea * u.abs() + a.abs() * eu + U32 * h.abs() + rounded(h)
    y = h @ wd.T
    val = {"y": y}
    err = {"y": eh @ wd.abs().T + (hidden + 2) * U32 * (h.abs() @ wd.abs().T) + rounded(y)}
    dh = dy @ wd
    edh = (d_out + 2) * U32 * (dy.abs() @ wd.abs())
    du, dg = dh * a, dh * u * s
    edu = edh * a.abs() + dh.abs() * ea + U32 * du.abs() + rounded(du)
    edg = edh * (u * s).abs() + dh.abs() * (eu * s.abs() + u.abs() * es) + 3 * U32 * dg.abs() \
        + rounded(dg)
    val["dx"] = dg @ wg + du @ wu
    err["dx"] = (edg + (2 * hidden + 3) * U32 * dg.abs()) @ wg.abs() \
        + (edu + (2 * hidden + 3) * U32 * du.abs()) @ wu.abs() + rounded(val["dx"])
    for name, d, e, other in (("dw_gate", dg, edg, x), ("dw_up", du, edu, x)):
        val[name] = d.T @ other
        err[name] = (e + (rows + 2) * U32 * d.abs()).T @ other.abs() + rounded(val[name])
    val["dw_down"] = dy.T @ h
    err["dw_down"] = dy.abs().T @ (eh + (rows + 2) * U32 * h.abs()) + rounded(val["dw_down"])
    return val, err


def outputs(x, wg, wu, wd, dy, act):
    leaves = [t.detach().requires_grad_(True) for t in (x, wg, wu, wd)]
    y = gated_feed_forward(*leaves, activation=act)
    grads = torch.autograd.grad(y, leaves, dy)
    return dict(zip(("y", "dx", "dw_gate", "dw_up", "dw_down"), (y.detach(), *grads)))


def check(got, val, err, dtype):
    # 16 bits: h's (or its gradient's) rounding and the output's, each half its
    # bound in the mean at most, and half as much again;
    # float32: sums of up to some thousand terms of random sign
    near = 1e-5 if dtype == torch.float32 else 1.5 * ROUND[dtype][0]
    for name, v in val.items():
        t = got[name]
        assert t.dtype == dtype and t.shape == v.shape
        d = (t.double() - v).abs()
        over = d - 1.02 * err[name]
        assert bool((over <= 0).all()), (name, float(over.max()), float(d.max()))
        rel = float(d.norm() / (v.norm() + 1e-300))
        assert rel <= near, (name, rel)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_block_against_64_bits(size, dtype):
    act = ACTS[sum(size) % 3]
    t = inputs(*size, dtype, seed=sum(size))
    check(outputs(*t, act), *formulas(*t, act), dtype)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_every_activation(act, dtype):
    t = inputs(200, 24, 72, 40, dtype, seed=5)
    check(outputs(*t, act), *formulas(*t, act), dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_strided_rows_and_leading_dimensions(dtype):
    x, wg, wu, wd, dy = inputs(6 * 35, 20, 48, 12, dtype, seed=2)
    val, err = formulas(x, wg, wu, wd, dy, "silu")
    wide = torch.full((6, 35, 29), float("nan"), dtype=dtype, device=DEV)
    wide[..., 3:23] = x.view(6, 35, 20)
    wide_dy = torch.full((6, 35, 13), float("nan"), dtype=dtype, device=DEV)
    wide_dy[..., 1:] = dy.view(6, 35, 12)
    wide_wg = torch.full((48, 21), float("nan"), dtype=dtype, device=DEV)
    wide_wg[:, 1:] = wg
    leaves = [wide[..., 3:23].detach().requires_grad_(True),
              wide_wg[:, 1:].detach().requires_grad_(True),
              wu.t().contiguous().t().detach().requires_grad_(True),
              wd.detach().requires_grad_(True)]
    y = gated_feed_forward(*leaves)
    assert y.shape == (6, 35, 12)
    grads = torch.autograd.grad(y, leaves, wide_dy[..., 1:])
    got = {"y": y.detach().reshape(-1, 12), "dx": grads[0].reshape(-1, 20), "dw_gate": grads[1],
           "dw_up": grads[2], "dw_down": grads[3]}
    check(got, val, err, dtype)
    # a row that is broadcast to many: its gradient is the rows' sum
    one = x[:1].detach().requires_grad_(True)
    y = gated_feed_forward(one.expand(9, 20), wg, wu, wd)
    (g1,) = torch.autograd.grad(y, one, torch.ones_like(y))
    alone = x[:1].detach().requires_grad_(True)
    (g2,) = torch.autograd.grad(gated_feed_forward(alone, wg, wu, wd), alone,
                                torch.ones((1, 12), dtype=dtype, device=DEV))
    tol = 9 * (2 ** -8 if dtype == torch.bfloat16 else 2 ** -10)
    assert torch.allclose(g1.float(), 9 * g2.float(), rtol=tol, atol=tol * float(g2.abs().max()))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_no_rows(dtype):
    _, wg, wu, wd, _ = inputs(1, 8, 16, 4, dtype)
    leaves = [torch.empty((0, 8), dtype=dtype, device=DEV, requires_grad=True)] + \
        [w.detach().requires_grad_(True) for w in (wg, wu, wd)]
    y = gated_feed_forward(*leaves)
    assert y.shape == (0, 4)
    for g, t in zip(torch.autograd.grad(y, leaves, torch.empty_like(y)), leaves):
        assert g.shape == t.shape and float(g.abs().sum()) == 0.0


@pytest.mark.parametrize("which", range(4))
def test_only_the_gradients_asked_for(which):
    t = inputs(150, 12, 40, 9, torch.float32, seed=8)
    val, err = formulas(*t, "silu")
    leaves = [v.detach().requires_grad_(i == which) for i, v in enumerate(t[:4])]
    y = gated_feed_forward(*leaves)
    (g,) = torch.autograd.grad(y, leaves[which], t[4])
    name = ("dx", "dw_gate", "dw_up", "dw_down")[which]
    assert bool(((g.double() - val[name]).abs() <= 1.02 * err[name]).all())


@pytest.mark.parametrize("size", [(90, 32, 64, 21), (40, 130, 70, 140)], ids=str)
@pytest.mark.parametrize("act", ACTS)
def test_gradient_against_differences(act, size):
    """Directional derivatives of sum(y * dy): the step 2^-6 leaves a
    truncation error of its square times third derivatives of order one, a
    rounding error of 2^-24 |y| |dy| / 2^-6 below it."""
    x, wg, wu, wd, dy = inputs(*size, torch.float32, seed=9)
    got = outputs(x, wg, wu, wd, dy, act)
    base = [x, wg, wu, wd]
    g = torch.Generator().manual_seed(3)
    step = 2.0 ** -6
    for i, name in enumerate(("dx", "dw_gate", "dw_up", "dw_down")):
        way = torch.randn(base[i].shape, generator=g).to(DEV)
        way = way / way.norm() * base[i].norm()
        ends = []
        for sign in (1, -1):
            moved = [t + sign * step * way if k == i else t for k, t in enumerate(base)]
            ends.append((gated_feed_forward(*moved, activation=act).double() * dy.double()).sum())
        numeric = float(ends[0] - ends[1]) / (2 * step)
        exact = float((got[name].double() * way.double()).sum())
        size_of = float(got[name].norm() * way.norm())
        assert abs(numeric - exact) <= 2e-3 * size_of, (name, numeric, exact)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_a_row_that_is_not_finite_stays_alone(dtype):
    """NaN and infinite features spoil their own outputs, no other row's."""
    x, wg, wu, wd, dy = inputs(200, 32, 64, 21, dtype, seed=4)
    clean = gated_feed_forward(x, wg, wu, wd)
    spoilt = x.clone()
    spoilt[17, 3] = float("nan")
    spoilt[90, 0] = float("inf")
    spoilt[199] = float("-inf")
    leaf = spoilt.requires_grad_(True)
    y = gated_feed_forward(leaf, wg, wu, wd)
    (dx,) = torch.autograd.grad(y, leaf, dy)
    bad = torch.zeros(200, dtype=torch.bool)
    bad[[17, 90, 199]] = True
    assert bool(y[17].isnan().all())
    assert torch.equal(y.detach()[~bad], clean[~bad])
    assert bool(dx[~bad].isfinite().all())
    assert not bool(y[90].isfinite().any()) and not bool(y[199].isfinite().any())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_far_arguments(dtype):
    """Gates far out on both sides: the activations' limits, no overflow."""
    for act, limits in (("silu", (0.0, 300.0)), ("gelu", (0.0, 300.0)), ("sigmoid", (0.0, 1.0))):
        for sign, a in zip((-1.0, 1.0), limits):
            x = torch.tensor([[300.0 * sign, 1.0]], dtype=dtype, device=DEV).requires_grad_(True)
            wg = torch.tensor([[1.0, 0.0]], dtype=dtype, device=DEV)
            wu = torch.tensor([[0.0, 1.0]], dtype=dtype, device=DEV)
            wd = torch.tensor([[1.0]], dtype=dtype, device=DEV)
            y = gated_feed_forward(x, wg, wu, wd, activation=act)
            assert float(y) == a
            (dx,) = torch.autograd.grad(y, x)
            slope = 1.0 if act != "sigmoid" and sign > 0 else 0.0
            assert dx.tolist() == [[slope, a]]


def test_same_bits_every_time_and_on_another_stream():
    t = inputs(5000, 32, 128, 64, torch.float32, seed=1)
    first = outputs(*t, "silu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = outputs(*t, "silu")
    torch.cuda.current_stream().wait_stream(side)
    for k in first:
        assert torch.equal(first[k], second[k]), k


def test_module_trains():
    block = GatedFeedForward(8, 32, 3, activation="gelu", seed=1)
    x = torch.randn((256, 8), generator=torch.Generator().manual_seed(0)).to(DEV)
    y = block(x)
    assert y.shape == (256, 3) and set(block.params) == {"w_gate", "w_up", "w_down"}
    y.square().mean().backward()
    assert all(p.grad is not None and bool(p.grad.isfinite().all()) for p in block.params.values())


def test_more_elements_than_32_bits_count():
    """x and its gradient of more than 2^32 elements, the hidden channels in two
    groups whose parts of dx are added up: rows at both ends and on both sides of
    the 2^31st and the 2^32nd element against the formulas."""
    if torch.cuda.mem_get_info()[0] < 100 << 30:
        pytest.skip("takes 100 GB of device memory")
    d_in, hidden = 128, 160
    rows = (1 << 32) // d_in + 3
    g = torch.Generator(device=DEV).manual_seed(6)
    x = torch.empty((rows, d_in), dtype=torch.bfloat16, device=DEV)
    for part in x.split(1 << 22):
        part.copy_(torch.randn(part.shape, generator=g, device=DEV))
    _, wg, wu, wd, _ = inputs(1, d_in, hidden, 1, torch.bfloat16, seed=6)
    dy = torch.ones((rows, 1), dtype=torch.bfloat16, device=DEV)
    x.requires_grad_(True)
    y = gated_feed_forward(x, wg, wu, wd)
    (dx,) = torch.autograd.grad(y, x, dy)
    picks = torch.tensor([0, 1, rows // 2 - 1, rows // 2, rows // 2 + 1, rows - 4, rows - 3,
                          rows - 2, rows - 1], device=DEV)
    val, err = formulas(x.detach()[picks], wg, wu, wd, dy[picks], "silu")
    got = {"y": y.detach()[picks], "dx": dx[picks]}
    check(got, {k: val[k] for k in got}, err, torch.bfloat16)
