"""Layer norm against its formulas in 64 bits, its gradients against differences, and
its layouts.

Each output is held to a first-order bound of what float32 arithmetic and the rounding
to the tensors' type can do, from the magnitudes of the terms (in float64 beside the
values).  With u = 2^-24 and a sum's chain of at most k = width + 8 additions:
  d = x - m0 for a rounded mean m0: u |d|, and the row's offset is known to
      e_off = k u mean|d|, so e_d = u |d| + e_off;  m0 itself is within
      |m0 - m| <= k u mean|x| of the mean, which enters |d|
  v = mean d^2 - off^2: e_v = (k + 3) u mean d^2 + 2 e_off mean|d|
  r = (v + eps)^-1/2: e_r = r (e_v r^2 / 2 + 4 u)
  h = d r, y = h w + b, and the gradient's sums likewise."""

import pytest
import torch

from mlx3d_amd.nn import LayerNorm, layer_norm

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = 2.0 ** -24
TYPES = (torch.float32, torch.bfloat16, torch.float16)
# half a step relative to the value, and half the smallest subnormal
ROUND = {torch.float32: (2.0 ** -24, 2.0 ** -150), torch.bfloat16: (2.0 ** -8, 2.0 ** -134),
         torch.float16: (2.0 ** -11, 2.0 ** -25)}

# one row, one column, no width a multiple of a vector, both sides of where a team of
# lanes, a wave and a workgroup hold a row in each type, and longer rows
SIZES = [(1, 1), (1, 32), (3, 2), (5, 3), (257, 7), (64, 8), (1000, 9), (33, 27), (2500, 32),
         (129, 48), (70, 65), (300, 96), (31, 127), (9, 256), (8, 257), (11, 512), (7, 513),
         (5, 1024), (6, 1025), (130, 1365), (4, 2048), (3, 2049), (5, 4096), (4, 4097), (3, 8192),
         (3, 8193), (2, 12289), (20_000, 5), (9000, 24)]


def inputs(rows, width, dtype, seed=0, offset=0.5, spread=1.0):
    g = torch.Generator().manual_seed(seed)

    def n(*s):
        return torch.randn(s, generator=g)

    x = (n(rows, width) * spread + offset) * (0.02 + 0.98 * torch.rand((rows, 1), generator=g))
    return [t.to(dtype).to(DEV) for t in (x, 1 + 0.2 * n(width), 0.2 * n(width), n(rows, width))]


def formulas(x, w, b, dy, eps):
    """Values in float64 and a bound of each output's error."""
    ulp, sub = ROUND[x.dtype]
    x, w, b, dy = (t.double() for t in (x, w, b, dy))
    rows, width = x.shape
    k = width + 8

    def mean(t):
        return t.mean(dim=1, keepdim=True)

    shift = k * U * mean(x.abs())             # of the rounded mean, inside |d|
    d = x - mean(x)
    size = d.abs() + shift
    e_off = k * U * mean(size)
    e_d = 2 * U * size + e_off
    var = mean(d * d)
    e_v = (k + 3) * U * mean(size * size) + 2 * e_off * mean(size) + shift * shift * k * U
    r = (var + eps) ** -0.5
    e_r = r * (0.5 * e_v * r * r + 4 * U)
    h = d * r
    e_h = e_d * r + size * e_r + U * h.abs()
    y = h * w + b
    g = dy * w
    mg, mgh = mean(g), mean(g * h)
    e_mg = (k + 2) * U * mean(g.abs())
    e_mgh = (k + 4) * U * mean(g.abs() * size) * r + mean(g.abs() * e_h)
    inner = g - mg - h * mgh
    e_in = U * g.abs() + e_mg + h.abs() * e_mgh + e_h * mgh.abs() + \
        3 * U * (g.abs() + mg.abs() + (h * mgh).abs())
    val = {"y": y, "dx": inner * r, "dw": (dy * h).sum(0), "db": dy.sum(0)}
    err = {"y": e_h * w.abs() + U * (h * w).abs() + U * y.abs(),
           "dx": e_in * r + inner.abs() * e_r + U * val["dx"].abs(),
           "dw": (dy.abs() * e_h).sum(0) + (rows + 2) * U * (dy * h).abs().sum(0),
           "db": (rows + 2) * U * dy.abs().sum(0)}
    return val, {name: 1.01 * e + ulp * val[name].abs() + sub for name, e in err.items()}


def outputs(x, w, b, dy, eps=1e-5):
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    y = layer_norm(*leaves, eps=eps)
    return dict(zip(("y", "dx", "dw", "db"), (y.detach(), *torch.autograd.grad(y, leaves, dy))))


def check(got, val, err, dtype):
    for name, t in got.items():
        assert t.dtype == dtype and t.shape == val[name].shape
        over = (t.double() - val[name]).abs() - err[name]
        assert bool((over <= 0).all()), (name, float(over.max()))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_against_64_bits(size, dtype):
    t = inputs(*size, dtype, seed=sum(size))
    check(outputs(*t), *formulas(*t, 1e-5), dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("size", [(5000, 1030), (1700, 2100), (1300, 4300), (700, 8100),
                                  (600, 8200), (9000, 520), (70_000, 96), (150_000, 3)], ids=str)
def test_workgroups_that_walk_many_rows(size, dtype):
    """More rows than teams at once, in each kind of team: several rounds a workgroup."""
    t = inputs(*size, dtype, seed=sum(size))
    check(outputs(*t), *formulas(*t, 1e-5), dtype)


@pytest.mark.parametrize("width", (27, 96, 700, 5000))
def test_far_from_zero(width):
    """Rows whose mean is a thousand times their spread keep the spread's digits."""
    t = inputs(40, width, torch.float32, seed=3, offset=1000.0)
    check(outputs(*t), *formulas(*t, 1e-5), torch.float32)


@pytest.mark.parametrize("eps", (1.2e-38, 1e-12, 1e-3, 10.0))
def test_eps(eps):
    t = inputs(50, 40, torch.float32, seed=4)
    check(outputs(*t, eps), *formulas(*t, eps), torch.float32)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("width", (1, 5, 32, 300, 9000))
def test_constant_rows(width, dtype):
    """Nothing varies: y is the bias, and dx stays finite."""
    _, w, b, dy = inputs(6, width, dtype)
    x = torch.tensor([[0.0], [1.0], [-3.5], [0.1], [60000.0], [1e-7]]).to(dtype).to(DEV)
    got = outputs(x.expand(6, width).contiguous(), w, b, dy)
    assert torch.equal(got["y"][0], b)
    # (x - m) is a rounding of the sum at most
    assert bool(((got["y"] - b).float().abs() <=
                 (width + 8) * U * x.float().abs() * 317 * w.float().abs()
                 + 2.0 ** -8 * b.float().abs()).all())
    assert all(bool(v.isfinite().all()) for v in got.values())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("width", (20, 333))
def test_strided_rows_and_leading_dimensions(width, dtype):
    x, w, b, dy = inputs(6 * 35, width, dtype, seed=2)
    val, err = formulas(x, w, b, dy, 1e-5)
    wide = torch.full((6, 35, width + 9), float("nan"), dtype=dtype, device=DEV)
    wide[..., 3:3 + width] = x.view(6, 35, width)
    wide_dy = torch.full((6, 35, width + 1), float("nan"), dtype=dtype, device=DEV)
    wide_dy[..., 1:] = dy.view(6, 35, width)
    long_w = torch.full((2 * width,), float("nan"), dtype=dtype, device=DEV)
    long_w[::2] = w
    odd_b = torch.full((width + 1,), float("nan"), dtype=dtype, device=DEV)
    odd_b[1:] = b
    leaves = [t.detach().requires_grad_(True) for t in (wide[..., 3:3 + width], long_w[::2],
                                                        odd_b[1:])]
    y = layer_norm(*leaves)
    assert y.shape == (6, 35, width) and y.is_contiguous()
    grads = torch.autograd.grad(y, leaves, wide_dy[..., 1:])
    got = {"y": y.detach().reshape(-1, width), "dx": grads[0].reshape(-1, width), "dw": grads[1],
           "db": grads[2]}
    check(got, val, err, dtype)


def test_other_orders():
    """Transposed inputs, one row for many (its gradient their sum), one value."""
    x, w, b, dy = inputs(24, 24, torch.float32, seed=6)
    val, err = formulas(x, w, b, dy, 1e-5)
    turned = x.t().contiguous().t().requires_grad_(True)
    y = layer_norm(turned, w, b)
    (dx,) = torch.autograd.grad(y, turned, dy.t().contiguous().t())
    check({"y": y.detach(), "dx": dx}, val, err, torch.float32)
    one = x[:1].detach().requires_grad_(True)
    (many,) = torch.autograd.grad(layer_norm(one.expand(9, 24), w, b).sum(), one)
    alone = x[:1].detach().requires_grad_(True)
    (once,) = torch.autograd.grad(layer_norm(alone, w, b).sum(), alone)
    # the same nine values' sum
    assert torch.allclose(many, 9 * once, rtol=9 * 2.0 ** -23, atol=0)
    scalar = layer_norm(x[0, :1])
    assert scalar.shape == (1,) and float(scalar) == 0.0


@pytest.mark.parametrize("with_weight", (False, True))
@pytest.mark.parametrize("with_bias", (False, True))
@pytest.mark.parametrize("size", ((70, 30), (9, 4500)), ids=str)
def test_without_weights(size, with_weight, with_bias):
    x, w, b, dy = inputs(*size, torch.float32, seed=7)
    one, zero = torch.ones_like(w), torch.zeros_like(b)
    val, err = formulas(x, w if with_weight else one, b if with_bias else zero, dy, 1e-5)
    leaves = [x.requires_grad_(True)] + [t.requires_grad_(True) for t, k in
                                         ((w, with_weight), (b, with_bias)) if k]
    y = layer_norm(x, w if with_weight else None, b if with_bias else None)
    names = ["dx"] + ["dw"] * with_weight + ["db"] * with_bias
    got = dict(zip(names, torch.autograd.grad(y, leaves, dy)))
    check({"y": y.detach(), **got}, val, err, torch.float32)


@pytest.mark.parametrize("which", range(3))
@pytest.mark.parametrize("size", ((150, 12), (40, 700), (10, 5000)), ids=str)
def test_only_the_gradient_asked_for(size, which):
    t = inputs(*size, torch.float32, seed=8)
    val, err = formulas(*t, 1e-5)
    leaves = [v.detach().requires_grad_(i == which) for i, v in enumerate(t[:3])]
    (g,) = torch.autograd.grad(layer_norm(*leaves), leaves[which], t[3])
    check({("dx", "dw", "db")[which]: g}, val, err, torch.float32)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_no_rows(dtype):
    _, w, b, _ = inputs(1, 8, dtype)
    leaves = [t.requires_grad_(True) for t in (torch.empty((0, 8), dtype=dtype, device=DEV), w, b)]
    y = layer_norm(*leaves)
    assert y.shape == (0, 8)
    for g, t in zip(torch.autograd.grad(y, leaves, torch.empty_like(y)), leaves):
        assert g.shape == t.shape and float(g.abs().sum()) == 0.0


@pytest.mark.parametrize("size", ((90, 21), (40, 260), (12, 4200)), ids=str)
def test_gradient_against_differences(size):
    """Directional derivatives of sum(y * dy) in steps of 2^-6 of the row's spread: a
    truncation of the step's square times third derivatives of order one, and a rounding
    of 2^-24 |y| |dy| / 2^-6 below it."""
    x, w, b, dy = inputs(*size, torch.float32, seed=9)
    x = x + torch.randn(x.shape, generator=torch.Generator().manual_seed(1)).to(DEV)
    got, base, step = outputs(x, w, b, dy), [x, w, b], 2.0 ** -6
    g = torch.Generator().manual_seed(3)
    for i, name in enumerate(("dx", "dw", "db")):
        way = torch.randn(base[i].shape, generator=g).to(DEV)
        way = way / way.norm() * base[i].norm() * (0.2 if i == 0 else 1.0)
        ends = []
        for sign in (1, -1):
            moved = [t + sign * step * way if k == i else t for k, t in enumerate(base)]
            ends.append((layer_norm(*moved).double() * dy.double()).sum())
        numeric = float(ends[0] - ends[1]) / (2 * step)
        exact = float((got[name].double() * way.double()).sum())
        assert abs(numeric - exact) <= 2e-3 * float(got[name].norm() * way.norm()), name


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("width", (6, 32, 500, 9000))
def test_a_row_that_is_not_finite_stays_alone(width, dtype):
    x, w, b, dy = inputs(40, width, dtype, seed=4)
    clean = outputs(x, w, b, dy)
    x[17, 3] = float("nan")
    x[20, 0] = float("inf")
    x[39] = float("-inf")
    got = outputs(x, w, b, dy)
    bad = torch.zeros(40, dtype=torch.bool)
    bad[[17, 20, 39]] = True
    for name in ("y", "dx"):
        assert bool(got[name][bad].isnan().all())
        assert torch.equal(got[name][~bad], clean[name][~bad])
    assert torch.equal(got["db"], clean["db"])


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16), ids=str)
@pytest.mark.parametrize("width", (6, 27, 32, 500, 1365, 9000))
def test_rows_beyond_the_range_of_squares(width, dtype):
    """Finite rows whose squares or whose sum float32 does not hold."""
    x, w, b, dy = inputs(40, width, dtype, seed=4)
    clean = outputs(x, w, b, dy)
    x[17] = (x[17].float() * 1e30).to(dtype)
    x[20] = (x[20].float() * 1e20).to(dtype)
    x[39] = 3e38
    got = outputs(x, w, b, dy)
    assert torch.equal(got["y"][17], b) and torch.equal(got["y"][20], b)
    assert not bool(got["dx"][[17, 20]].any())
    assert bool(got["y"][39].isnan().all()) and bool(got["dx"][39].isnan().all())
    rest = [i for i in range(39) if i not in (17, 20)]
    for name in ("y", "dx"):
        assert torch.equal(got[name][rest], clean[name][rest])
    assert torch.equal(got["db"], clean["db"])


def test_same_bits_every_time_and_on_another_stream():
    t = inputs(5000, 48, torch.float32, seed=1)
    first = outputs(*t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = outputs(*t)
    torch.cuda.current_stream().wait_stream(side)
    for k in first:
        assert torch.equal(first[k], second[k]), k


def test_module():
    norm = LayerNorm(24, eps=1e-4)
    assert set(norm.params) == {"weight", "bias"}
    x, _, _, dy = inputs(64, 24, torch.float32)
    one, zero = (norm.params[k].detach() for k in ("weight", "bias"))
    val, err = formulas(x, one, zero, dy, 1e-4)
    y = norm(x)
    y.backward(dy)
    check({"y": y.detach(), "dw": norm.params["weight"].grad, "db": norm.params["bias"].grad},
          val, err, torch.float32)


def test_more_elements_than_32_bits_count():
    """Rows at both ends and around the 2^31st and the 2^32nd element."""
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("takes 60 GB of device memory")
    width = 129
    rows = (1 << 32) // width + 5
    g = torch.Generator(device=DEV).manual_seed(6)
    x = torch.empty((rows, width), dtype=torch.bfloat16, device=DEV)
    for part in x.split(1 << 22):
        part.copy_(torch.randn(part.shape, generator=g, device=DEV))
    _, w, b, _ = inputs(1, width, torch.bfloat16, seed=6)
    x.requires_grad_(True)
    y = layer_norm(x, w, b)
    (dx,) = torch.autograd.grad(y, x, x.detach())
    half = (1 << 31) // width
    picks = torch.tensor([0, 1, half - 1, half, half + 1, rows - 6, rows - 5, rows - 2, rows - 1],
                         device=DEV)
    chosen = x.detach()[picks]
    val, err = formulas(chosen, w, b, chosen, 1e-5)
    check({"y": y.detach()[picks], "dx": dx[picks]}, val, err, torch.bfloat16)
