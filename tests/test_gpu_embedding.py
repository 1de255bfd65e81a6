"""Table lookups and the table's gradient against 64 bits, at the counts and
distributions where the sort, its tiles and their joins change."""

import pytest
import torch

from mlx3d_amd.nn import Embedding, embedding

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = 2.0 ** -24
TYPES = (torch.float32, torch.bfloat16, torch.float16)
# half a step relative to the value, and half the smallest subnormal
ROUND = {torch.float32: (2.0 ** -24, 2.0 ** -150), torch.bfloat16: (2.0 ** -8, 2.0 ** -134),
         torch.float16: (2.0 ** -11, 2.0 ** -25)}


def spread(how, count, rows, g):
    """Indices of one kind."""
    if how == "even":
        return torch.randint(0, rows, (count,), generator=g)
    if how == "one":  # all of one row, the last
        return torch.full((count,), rows - 1)
    if how == "few":  # popular ones, and many without a token
        return (rows * torch.rand((count,), generator=g) ** 4).long().clamp_(max=rows - 1)
    if how == "outside":  # half of them name no row
        k = torch.randint(-rows - 3, rows + 3, (count,), generator=g)
        return torch.where(torch.rand((count,), generator=g) < 0.5, k, k.abs())
    if how == "none":
        return torch.full((count,), -1)
    return torch.arange(count) % rows  # "turns"


def inputs(count, rows, width, dtype, how="even", seed=0, index=torch.int64):
    g = torch.Generator().manual_seed(seed)
    k = spread(how, count, rows, g).to(index)
    table = torch.randn((rows, width), generator=g).to(dtype)
    dy = torch.randn((count, width), generator=g).to(dtype)
    return k.to(DEV), table.to(DEV), dy.to(DEV)


def formulas(k, table, dy, scale):
    """Values in float64, and bounds: a float32 product and a rounding; for the gradient
    a chain of at most as many additions as the row has tokens."""
    ulp, sub = ROUND[table.dtype]
    k = k.long().reshape(-1)
    there = (k >= 0) & (k < table.shape[0])
    safe = torch.where(there, k, 0)
    y = torch.where(there[:, None], table.double()[safe] * scale, 0.0)
    told = torch.where(there[:, None], dy.reshape(len(k), -1).double(), 0.0)
    zero = torch.zeros(table.shape, dtype=torch.float64, device=DEV)
    grad = zero.index_add(0, safe, told) * scale
    size = zero.index_add(0, safe, told.abs()) * abs(scale)
    n = torch.zeros(len(table), dtype=torch.float64, device=DEV).index_add(0, safe, there.double())
    val = {"y": y, "grad": grad}
    err = {"y": U * y.abs() + ulp * y.abs() + sub,
           "grad": (n[:, None] + 1) * U * size + ulp * grad.abs() + sub}
    # the scale itself is rounded to float32
    return val, {name: e * 1.01 + U * val[name].abs() for name, e in err.items()}


def outputs(k, table, dy, scale=1.0):
    leaf = table.detach().requires_grad_(True)
    y = embedding(k, leaf, scale=scale)
    return {"y": y.detach(), "grad": torch.autograd.grad(y, leaf, dy)[0]}


def check(got, val, err, dtype):
    for name, t in got.items():
        assert t.dtype == dtype
        over = (t.double().reshape(val[name].shape) - val[name]).abs() - err[name]
        assert over.numel() == 0 or bool((over <= 0).all()), (name, float(over.max()))


# one token; both sides of a tile of 64, of a chunk of 4096; rows on both sides of a
# pass's digit of 8 bits, and more passes; widths that fill no vector, and wide ones
SIZES = [(1, 1, 1), (1, 4096, 64), (2, 3, 5), (63, 7, 4), (64, 256, 9), (65, 257, 32), (129, 2, 3),
         (1000, 100, 27), (4095, 300, 8), (4096, 17, 33), (4097, 70_000, 7), (5000, 1, 16),
         (9001, 65_536, 12), (300, 65_537, 130), (700, 20, 513), (33, 5, 2049), (20_000, 1000, 48),
         (100_003, 201, 6), (70_000, 1 << 24, 1), (8205, 5000, 100)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_against_64_bits(size, dtype):
    how = ("even", "few", "turns", "outside")[sum(size) % 4]
    t = inputs(*size, dtype, how, seed=sum(size),
               index=torch.int32 if size[0] % 2 else torch.int64)
    check(outputs(*t, 1.5), *formulas(*t, 1.5), dtype)


@pytest.mark.parametrize("how", ("even", "one", "few", "outside", "none", "turns"))
@pytest.mark.parametrize("size", ((500, 40, 20), (30_000, 1000, 32), (64 * 64, 129, 64)), ids=str)
def test_every_distribution(size, how):
    t = inputs(*size, torch.float32, how, seed=3)
    check(outputs(*t), *formulas(*t, 1.0), torch.float32)


def test_a_row_that_nearly_every_token_names():
    """Half a million terms: sums stay as exact as a tile's and a join's chains (their
    errors of random sign, far below the bound of one chain)."""
    k, table, dy = inputs(500_001, 50, 24, torch.float32, "few", seed=5)
    k[::2] = 11
    got = outputs(k, table, dy)
    val, err = formulas(k, table, dy, 1.0)
    check(got, val, err, torch.float32)
    assert float((got["grad"].double() - val["grad"]).norm() / val["grad"].norm()) < 1e-6


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_a_scale_of_one_copies_bits(dtype):
    k, table, dy = inputs(300, 40, 21, dtype)
    table[3, 2] = float("inf")
    table[4, 0] = float("nan")
    y = embedding(k, table)
    assert torch.equal(y.nan_to_num(nan=7.0), table[k].nan_to_num(nan=7.0))


def test_indices_outside():
    k = torch.tensor([0, -1, 3, 4, 2, -2 ** 31, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    far = torch.tensor([0, -1, 3, 2 ** 32, 2, -2 ** 63, 2 ** 63 - 1], device=DEV)
    table = torch.arange(1, 9, dtype=torch.float32, device=DEV).view(4, 2).requires_grad_(True)
    dy = torch.ones((7, 2), device=DEV)
    dy[1] = float("nan")  # of a token that names no row: reaches nothing
    for index in (k, far):
        y = embedding(index, table, scale=2.0)
        assert y.tolist() == [[2, 4], [0, 0], [14, 16], [0, 0], [10, 12], [0, 0], [0, 0]]
        (grad,) = torch.autograd.grad(y, table, dy)
        assert grad.tolist() == [[2, 2], [0, 0], [2, 2], [2, 2]]


def test_a_gradient_that_is_not_finite_stays_in_its_row():
    k, table, dy = inputs(5000, 30, 20, torch.float32, "turns")
    clean = outputs(k, table, dy)["grad"]
    dy[7] = float("nan")
    got = outputs(k, table, dy)["grad"]
    assert bool(got[7].isnan().all())
    keep = torch.arange(30, device=DEV) != 7
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_strides_and_shapes(dtype):
    k, table, dy = inputs(6 * 35, 50, 20, dtype, "outside", seed=2)
    val, err = formulas(k, table, dy, 1.0)
    wide = torch.full((50, 29), float("nan"), dtype=dtype, device=DEV)
    wide[:, 3:23] = table
    wide_dy = torch.full((6, 35, 23), float("nan"), dtype=dtype, device=DEV)
    wide_dy[..., 1:21] = dy.view(6, 35, 20)
    strided = torch.stack((k, k + 1), dim=1)[:, 0].view(6, 35)
    for leaf in (wide[:, 3:23].detach(), table.t().contiguous().t().detach()):
        leaf.requires_grad_(True)
        y = embedding(strided, leaf)
        assert y.shape == (6, 35, 20) and y.is_contiguous()
        (grad,) = torch.autograd.grad(y, leaf, wide_dy[..., 1:21])
        assert grad.shape == (50, 20)
        check({"y": y.detach(), "grad": grad}, val, err, dtype)
    one = embedding(k[0], table)
    assert one.shape == (20,) and torch.equal(one, embedding(k[:1], table)[0])
    # a broadcast gradient
    leaf = table.detach().requires_grad_(True)
    (grad,) = torch.autograd.grad(embedding(k, leaf).float().sum(), leaf)
    val, err = formulas(k, table, torch.ones_like(dy), 1.0)
    check({"grad": grad}, val, err, dtype)


def test_no_tokens():
    table = torch.ones((5, 3), device=DEV, requires_grad=True)
    y = embedding(torch.empty((0, 2), dtype=torch.int64, device=DEV), table)
    assert y.shape == (0, 2, 3)
    (grad,) = torch.autograd.grad(y, table, torch.empty_like(y))
    assert grad.shape == (5, 3) and float(grad.abs().sum()) == 0.0


def test_gradient_against_differences():
    """The lookup is linear: a step of 1 along a direction changes sum(y * dy) by the
    gradient's product with it, up to the sums' rounding."""
    k, table, dy = inputs(3000, 60, 17, torch.float32, "few", seed=4)
    got = outputs(k, table, dy, 0.5)["grad"].double()
    way = torch.randn(table.shape, generator=torch.Generator().manual_seed(1)).to(DEV)
    ends = [(embedding(k, t, 0.5).double() * dy.double()).sum() for t in (table + way, table - way)]
    size = (embedding(k, table.abs() + way.abs(), 0.5).double() * dy.double().abs()).sum()
    assert abs(float((ends[0] - ends[1]) / 2 - (got * way.double()).sum())) <= 1e-6 * float(size)


def test_same_bits_every_time_and_on_another_stream():
    t = inputs(50_000, 300, 32, torch.float32, "few", seed=1)
    first = outputs(*t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = outputs(*t)
    torch.cuda.current_stream().wait_stream(side)
    for name in first:
        assert torch.equal(first[name], second[name])


def test_module():
    table = Embedding(300, 24, scale=4.0, seed=1)
    k, _, dy = inputs(2000, 300, 24, torch.float32)
    y = table(k)
    assert abs(float(y.detach().std()) - 1.0) < 0.05
    y.backward(dy)
    val, err = formulas(k, table.params["table"].detach(), dy, 4.0)
    check({"y": y.detach(), "grad": table.params["table"].grad}, val, err, torch.float32)


def test_more_elements_than_32_bits_count():
    """Outputs, gradients and a table of more than 2^32 elements."""
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("takes 80 GB of device memory")
    width = 1025
    rows = (1 << 32) // width + 3
    g = torch.Generator(device=DEV).manual_seed(2)
    table = torch.empty((rows, width), dtype=torch.bfloat16, device=DEV)
    for part in table.split(1 << 19):
        part.copy_(torch.randn(part.shape, generator=g, device=DEV))
    k = torch.randperm(rows, generator=g, device=DEV)
    k[5] = k[rows - 1]
    table.requires_grad_(True)
    y = embedding(k, table)
    (grad,) = torch.autograd.grad(y, table, y.detach())
    half = (1 << 31) // width
    picks = torch.tensor([0, 4, 6, half - 1, half, half + 1, rows - 3, rows - 2], device=DEV)
    assert torch.equal(y.detach()[picks], table.detach()[k[picks]])
    assert torch.equal(grad[k[picks]], table.detach()[k[picks]])
    assert torch.equal(grad[k[5]], (2 * table.detach()[k[5]].float()).to(torch.bfloat16))


def test_rows_of_a_million_columns():
    """More column blocks and tokens than a launch holds: workgroups walk on."""
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("takes 60 GB of device memory")
    width, count = 1 << 20, 16_500
    g = torch.Generator(device=DEV).manual_seed(3)
    table = torch.randn((7, width), generator=g, device=DEV).to(torch.bfloat16)
    k = torch.randint(-1, 7, (count,), generator=g, device=DEV)
    y = embedding(k, table)
    for i in (0, 1, 16_383, 16_384, 16_385, count - 1):
        want = table[k[i]] if int(k[i]) >= 0 else torch.zeros_like(table[0])
        assert torch.equal(y[i], want)
    named = (k >= 0).sum()
    assert int((y[:, 0] != 0).sum()) == int(named) and int((y[:, -1] != 0).sum()) == int(named)


@pytest.mark.parametrize("mode", (torch.no_grad, torch.inference_mode))
def test_without_a_graph(mode):
    k, table, _ = inputs(40, 9, 12, torch.float32)
    want = embedding(k, table)
    with mode():
        y = embedding(k, table.requires_grad_(True) if mode is torch.no_grad else table)
        assert not y.requires_grad and torch.equal(y, want)
