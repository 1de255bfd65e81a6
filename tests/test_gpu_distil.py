"""The distillation loss and its gradient against the definition in 64 bits,
against differences, and at the edges: absent entries, empty rows, masked and
infinite logits, columns named twice, long and short vocabularies."""

import math

import pytest
import torch

from mlx3d_amd.losses import distillation_loss, distillation_value_and_grad

pytestmark = pytest.mark.gpu

DEV = "cuda"
U32 = 2.0 ** -24
ROUND = {torch.float32: (U32, 2.0 ** -149), torch.bfloat16: (2.0 ** -8, 2.0 ** -134),
         torch.float16: (2.0 ** -11, 2.0 ** -25)}
TYPES = (torch.float32, torch.bfloat16, torch.float16)
TEACHERS = ("logits", "log_probs")

# (rows, vocab, top)
SIZES = [(1, 1, 1), (3, 2, 2), (64, 21, 3), (65, 33, 5), (130, 150, 8), (17, 64, 64),
         (1000, 7, 4), (9, 1201, 10), (5, 2048, 32), (5, 2049, 33), (4, 4097, 100),
         (3, 8193, 7), (2, 50001, 256), (1, 200003, 64), (70, 300, 256)]


def inputs(rows, vocab, top, dtype, teacher, seed=0, absent=True):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn((rows, vocab), generator=g) * 3).to(dtype)
    scores = torch.rand((rows, vocab), generator=g)
    values, index = torch.topk(scores, top, dim=1)
    values = values * 6
    if teacher == "log_probs":
        mass = 0.3 + 0.69 * torch.rand((rows, 1), generator=g)
        values = torch.log_softmax(values, 1) + torch.log(mass)
    if absent and rows > 2:
        drop = torch.rand((rows, top), generator=g) < 0.2
        index[drop] = torch.randint(-3, 0, (int(drop.sum()),), generator=g)
        index[1, 0] = vocab  # one past the end
        values[1, 0] = float("nan")
        index[rows // 2] = -1
        values[2, top - 1] = -math.inf
    return logits.to(DEV), values.to(DEV), index.to(DEV)


def definition(logits, values, index, temp, teacher):
    """Each row's loss and gradient in float64, row by row, and the bound of
    their float32 evaluation."""
    rows, vocab = logits.shape
    losses, grads, loss_tol, grad_tol, active = [], [], [], [], []
    for s, v, i in zip(logits.double().cpu(), values.double().cpu(), index.cpu()):
        keep = [k for k in range(len(i)) if 0 <= int(i[k]) < vocab and v[k] != -math.inf]
        active.append(bool(keep))
        if not keep:
            losses.append(torch.zeros((), dtype=torch.float64))
            grads.append(torch.zeros(vocab, dtype=torch.float64))
            loss_tol.append(torch.zeros((), dtype=torch.float64))
            grad_tol.append(torch.zeros(vocab, dtype=torch.float64))
            continue
        i, v = i[keep].long(), v[keep]
        z = s / temp
        log_q = torch.log_softmax(z, 0)
        q = log_q.exp()
        log_p = torch.log_softmax(v / temp, 0) if teacher == "logits" else v
        p = log_p.exp()
        term = torch.where(p > 0, p * (log_p - log_q[i]), torch.zeros(()).double())
        loss = term.sum()
        named = torch.zeros(vocab, dtype=torch.bool)
        named[i] = True
        total = p.sum()
        grad = torch.zeros(vocab, dtype=torch.float64).index_add_(0, i, -p)
        size = torch.zeros(vocab, dtype=torch.float64).index_add_(0, i, p)
        scale = (p * (log_p.abs() + log_q[i].abs())).nan_to_num(0).sum() + 1
        if teacher == "log_probs" and bool((~named & (s > -math.inf)).any()):
            r = max(0.0, 1.0 - float(total))
            log_big = torch.logsumexp(log_q[~named], 0)
            if r > 0:
                loss = loss + r * (math.log(r) - log_big)
                scale = scale + (r + 8) * (abs(math.log(r)) + abs(float(log_big)))
            share = torch.where(named, torch.zeros(()).double(), (log_q - log_big).exp())
            grad = grad - r * share
            total = total + r
            size = size + (r + 8) * share
        grad = temp * (grad + total * q)
        # a term's error: its exponent's rounding (4 |z - max|), its sums'
        # (a lane adds vocab / 32 terms at most, then a tree), 64 for the rest
        finite = z[z > -math.inf]
        c = 64 + 4 * float(finite.max() - finite.min()) + vocab / 32
        losses.append(loss * temp * temp)
        grads.append(grad)
        loss_tol.append(temp * temp * U32 * c * scale)
        grad_tol.append(temp * U32 * c * (size + total * q))
    return (torch.stack(losses), torch.stack(grads), torch.stack(loss_tol), torch.stack(grad_tol),
            torch.tensor(active))


def near_rows(got, want, tol, dtype=None):
    got = got.double().cpu()
    r, sub = ROUND[dtype] if dtype else (U32, 0.0)
    over = (got - want).abs() - (1.02 * tol + r * want.abs() + sub)
    assert bool((over <= 0).all()), (float(over.max()), float((got - want).abs().max()))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("teacher", TEACHERS)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_against_64_bits(size, teacher, dtype):
    temp = (1.0, 2.0, 0.5)[sum(size) % 3]
    logits, values, index = inputs(*size, dtype, teacher, seed=sum(size))
    loss, grad, loss_tol, grad_tol, active = definition(logits, values, index, temp, teacher)
    leaf = logits.detach().requires_grad_(True)
    got = distillation_loss(leaf, values, index, temperature=temp, teacher=teacher,
                            reduction="none")
    assert got.shape == (size[0],) and got.dtype == torch.float32
    near_rows(got.detach(), loss, loss_tol)
    w = 0.5 + torch.rand(size[0], generator=torch.Generator().manual_seed(1))
    (g,) = torch.autograd.grad(got, leaf, w.to(DEV))
    wd = w.double()[:, None]
    near_rows(g, grad * wd, grad_tol * wd, dtype)
    # the mean over the rows that have entries, in both forms; the sum
    n = max(1, int(active.sum()))
    mean = distillation_loss(leaf, values, index.int(), temperature=temp, teacher=teacher)
    near_rows(mean.detach(), loss.sum() / n, loss_tol.sum() / n)
    (g,) = torch.autograd.grad(mean, leaf)
    near_rows(g, grad / n, grad_tol / n, dtype)
    value, g2 = distillation_value_and_grad(logits, values, index, temperature=temp,
                                            teacher=teacher, scale=3.0)
    near_rows(value, 3 * loss.sum() / n, 3 * loss_tol.sum() / n)
    near_rows(g2, 3 * grad / n, 3 * grad_tol / n, dtype)
    value, g3 = distillation_value_and_grad(logits, values, index, temperature=temp,
                                            teacher=teacher, reduction="sum")
    near_rows(value, loss.sum(), loss_tol.sum())
    near_rows(g3, grad, grad_tol, dtype)
    total = distillation_loss(logits, values, index, temperature=temp, teacher=teacher,
                              reduction="sum")
    assert float(total) == float(value)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("teacher", TEACHERS)
@pytest.mark.parametrize("size", [(33, 11, 5), (50, 23, 8), (7, 41, 6), (70, 110, 13), (9, 300, 30),
                                  (5, 800, 70), (3, 2037, 128)], ids=str)
def test_two_entries_a_lane(size, teacher, dtype):
    test_against_64_bits(size, teacher, dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("vocab", [30, 5000])
@pytest.mark.parametrize("teacher", TEACHERS)
def test_masked_columns_and_rows(vocab, dtype, teacher):
    """Columns at -inf and at the type's lowest value; rows without entries
    whose logits are NaN and infinite."""
    logits, values, index = inputs(40, vocab, 5, dtype, teacher, seed=3)
    logits[:, 0] = -math.inf
    logits[:, 1] = torch.finfo(dtype).min
    index = torch.where((index == 0) | (index == 1), torch.full_like(index, 2), index)
    loss, grad, loss_tol, grad_tol, _ = definition(
        torch.where(logits == torch.finfo(dtype).min, torch.full_like(logits, -math.inf), logits),
        values, index, 1.0, teacher)
    empty = (index < 0).all(1) | (values == -math.inf).all(1)
    assert bool(empty[20])
    logits[20] = math.nan
    logits[20, 3] = math.inf
    values[20] = math.nan
    got, g = distillation_value_and_grad(logits, values, index, teacher=teacher, reduction="sum")
    near_rows(got, loss.sum(), loss_tol.sum())
    near_rows(g, grad, grad_tol, dtype)
    assert float(g[20].abs().sum()) == 0.0
    assert float(g[:20, :2].abs().sum()) == 0.0
    each = distillation_loss(logits, values, index, teacher=teacher, reduction="none")
    assert float(each[20]) == 0.0


@pytest.mark.parametrize("vocab", [30, 5000])
def test_a_named_column_that_is_ruled_out(vocab):
    """A student that gives a named column no mass: infinite loss, finite gradient."""
    logits, values, index = inputs(8, vocab, 4, torch.float32, "logits", seed=5, absent=False)
    logits[3, index[3, 1]] = -math.inf
    leaf = logits.requires_grad_(True)
    loss = distillation_loss(leaf, values, index, reduction="none")
    assert float(loss[3]) == math.inf and bool(loss[[0, 1, 2, 4, 5, 6, 7]].isfinite().all())
    (g,) = torch.autograd.grad(loss.sum(), leaf)
    p = torch.softmax(values[3].double(), 0)
    q = torch.softmax(logits[3].detach().double(), 0)
    want = q.index_add(0, index[3], -p)
    assert bool(((g[3].double() - want).abs() <= 1e-5).all())


@pytest.mark.parametrize("vocab", [30, 5000])
@pytest.mark.parametrize("teacher", TEACHERS)
def test_nan_spoils_its_own_row(vocab, teacher):
    logits, values, index = inputs(9, vocab, 4, torch.float32, teacher, seed=6, absent=False)
    clean = distillation_value_and_grad(logits, values, index, teacher=teacher, reduction="sum")[1]
    logits[2, 5] = math.nan
    values[7, 1] = math.nan
    each = distillation_loss(logits, values, index, teacher=teacher, reduction="none")
    g = distillation_value_and_grad(logits, values, index, teacher=teacher, reduction="sum")[1]
    for row in range(9):
        if row in (2, 7):
            assert math.isnan(float(each[row])) and bool(g[row].isnan().any())
        else:
            assert math.isfinite(float(each[row])) and torch.equal(g[row], clean[row])


@pytest.mark.parametrize("vocab", [12, 40, 9000])
@pytest.mark.parametrize("teacher", TEACHERS)
def test_columns_named_twice(vocab, teacher):
    logits, values, index = inputs(6, vocab, 6, torch.float32, teacher, seed=7, absent=False)
    index[:, 3] = index[:, 0]
    index[:, 5] = index[:, 0]
    loss, grad, loss_tol, grad_tol, _ = definition(logits, values, index, 1.0, teacher)
    got, g = distillation_value_and_grad(logits, values, index, teacher=teacher, reduction="sum")
    near_rows(got, loss.sum(), loss_tol.sum())
    near_rows(g, grad, grad_tol, torch.float32)


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16), ids=str)
def test_far_logits(dtype):
    """The rest far below the entries, and the entries far below the rest."""
    for vocab in (20, 6000):
        for low in (True, False):
            logits, values, index = inputs(5, vocab, 3, dtype, "log_probs", seed=8, absent=False)
            shift = torch.zeros_like(logits).scatter_(1, index, 200.0 if low else -200.0)
            logits = logits + shift
            want = definition(logits, values, index, 1.0, "log_probs")
            got, g = distillation_value_and_grad(logits, values, index, teacher="log_probs",
                                                 reduction="sum")
            near_rows(got, want[0].sum(), want[2].sum())
            near_rows(g, want[1], want[3], dtype)


def test_the_whole_mass_and_the_whole_vocabulary():
    """Log-probabilities that sum to one, and entries for every column: the
    plain divergence, no bucket."""
    g = torch.Generator().manual_seed(2)
    logits = torch.randn((50, 16), generator=g).to(DEV)
    lp = torch.log_softmax(torch.randn((50, 16), generator=g), 1).to(DEV)
    index = torch.arange(16, device=DEV).expand(50, 16)
    got = distillation_loss(logits, lp, index, teacher="log_probs", reduction="none")
    lp64 = lp.double()
    want = (lp64.exp() * (lp64 - torch.log_softmax(logits.double(), 1))).sum(1)
    assert bool(((got.double() - want).abs() <= 200 * U32 * (1 + want.abs())).all())


@pytest.mark.parametrize("vocab", [21, 4500])
def test_gradient_against_differences(vocab):
    """Central differences of the float32 sum: step 2^-5, truncation of its
    square times third derivatives below one."""
    for teacher in TEACHERS:
        logits, values, index = inputs(12, vocab, 5, torch.float32, teacher, seed=4)
        _, g = distillation_value_and_grad(logits, values, index, temperature=1.5,
                                           teacher=teacher, reduction="sum")
        way = torch.randn(logits.shape, generator=torch.Generator().manual_seed(0)).to(DEV)
        step = 2.0 ** -5
        ends = [distillation_loss(logits + s * step * way, values, index, temperature=1.5,
                                  teacher=teacher, reduction="none").double().sum()
                for s in (1, -1)]
        numeric = float(ends[0] - ends[1]) / (2 * step)
        exact = float((g.double() * way.double()).sum())
        assert abs(numeric - exact) <= 2e-3 * float(g.norm() * way.norm()), (numeric, exact)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("vocab", [21, 150, 5000])
def test_strided_logits_and_leading_dimensions(vocab, dtype):
    logits, values, index = inputs(24, vocab, 5, dtype, "logits", seed=9)
    want, g_want = distillation_value_and_grad(logits, values, index)
    for extra, first in ((1, 0), (3, 1), (8, 8)):
        wide = torch.full((4, 6, vocab + extra), math.nan, dtype=dtype, device=DEV)
        view = wide[..., first:first + vocab] if first + vocab <= vocab + extra else None
        view.copy_(logits.view(4, 6, vocab))
        got, g = distillation_value_and_grad(view, values.view(4, 6, 5), index.view(4, 6, 5))
        assert g.shape == (4, 6, vocab)
        assert torch.equal(got, want) and torch.equal(g.reshape(24, vocab), g_want)
    turned = logits.t().contiguous().t()
    got, g = distillation_value_and_grad(turned, values.double(), index)
    assert torch.equal(got, want) and torch.equal(g, g_want)
    # one row shared by many: its gradient is their sum
    leaf = logits[:1].float().detach().requires_grad_(True)
    loss = distillation_loss(leaf.expand(24, vocab), values, index, reduction="sum")
    (g,) = torch.autograd.grad(loss, leaf)
    parts = distillation_value_and_grad(leaf.detach().expand(24, vocab), values, index,
                                        reduction="sum")[1].double().sum(0)
    assert bool(((g[0].double() - parts).abs() <= 24 * 24 * U32).all())


def test_no_rows_and_no_entries():
    empty = torch.empty((0, 7), device=DEV, requires_grad=True)
    none = torch.empty((0, 2), device=DEV)
    for reduction in ("none", "sum", "mean"):
        loss = distillation_loss(empty, none, none.long(), reduction=reduction)
        assert loss.numel() == (0 if reduction == "none" else 1) and float(loss.sum()) == 0.0
        (g,) = torch.autograd.grad(loss.sum(), empty)
        assert g.shape == (0, 7)
    logits = torch.full((5, 7), math.nan, device=DEV)
    index = torch.full((5, 2), -1, device=DEV)
    loss, g = distillation_value_and_grad(logits, torch.zeros((5, 2), device=DEV), index)
    assert float(loss) == 0.0 and float(g.abs().sum()) == 0.0


def test_same_bits_every_time_and_on_another_stream():
    for vocab in (21, 20000):
        logits, values, index = inputs(300, vocab, 5, torch.bfloat16, "log_probs", seed=1)
        first = distillation_value_and_grad(logits, values, index, teacher="log_probs")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            second = distillation_value_and_grad(logits, values, index, teacher="log_probs")
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_more_logits_than_32_bits_count():
    """Offsets past 2^31 elements: the last rows of a large table."""
    rows, vocab = 11_000_000, 200
    logits = torch.zeros((rows, vocab), dtype=torch.bfloat16, device=DEV)
    values = torch.zeros((rows, 1), device=DEV)
    index = torch.full((rows, 1), -1, dtype=torch.int32, device=DEV)
    index[-2:] = 3
    logits[-1, 3] = 5.0
    loss, g = distillation_value_and_grad(logits, values, index)
    want = [math.log(vocab), math.log(199 + math.exp(5.0)) - 5.0]
    assert abs(float(loss) - sum(want) / 2) < 1e-5
    assert abs(float(g[-2, 3]) - (1 / vocab - 1) / 2) < 2e-3
    assert float(g[:-2].float().abs().max()) == 0.0


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("teacher", TEACHERS)
@pytest.mark.parametrize("vocab", (1, 2, 3, 5, 7))
def test_rows_that_begin_and_end_between_pieces(vocab, teacher, dtype):
    """Short rows in a buffer at every offset from a 16-byte boundary, with last
    tiles of a row or two that share their 16 bytes with the tile before.  By
    whole words off, the bits of the same rows at a boundary; else rows begin
    inside other words and their sums take another order: the definition."""
    top = min(vocab, 2)
    size = torch.empty((), dtype=dtype).element_size()
    for rows in (1, 2, 15, 16, 17, 18, 33, 49, 1025):
        logits, values, index = inputs(rows, vocab, top, dtype, teacher, seed=rows)
        want = distillation_value_and_grad(logits.clone(), values, index, teacher=teacher,
                                           reduction="sum")
        if rows < 50:
            loss, grad, loss_tol, grad_tol, _ = definition(logits, values, index, 1.0, teacher)
        for offset in range(1, 16 // size):
            buf = torch.full((offset + rows * vocab + 16,), float("nan"), dtype=dtype, device=DEV)
            view = buf[offset:offset + rows * vocab].view(rows, vocab)
            view.copy_(logits)
            got = distillation_value_and_grad(view, values, index, teacher=teacher,
                                              reduction="sum")
            if offset * size % 4 == 0:
                for a, b in zip(got, want):
                    assert torch.equal(a, b), (rows, offset)
            elif rows < 50:
                near_rows(got[0], loss.sum(), loss_tol.sum())
                near_rows(got[1], grad, grad_tol, dtype)
