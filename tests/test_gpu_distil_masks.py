"""The distillation loss where a finite value stands for a mask: whole segments,
everything outside the entries, whole rows, named columns and the teacher's own
values at the type's lowest value, -1e9, -1e10 and -1e30.

A masked column's power is 0 or, where only masks are left, the power of an
exact difference of equal values, so the bounds are those of ordinary rows: 64
float32 roundings, four for each unit of an exponent that still counts (above
-110), a sum of vocab / 32 terms on a lane."""

import math

import pytest
import torch

from mlx3d_amd.losses import distillation_loss, distillation_value_and_grad

pytestmark = pytest.mark.gpu

DEV = "cuda"
U32 = 2.0 ** -24
F32_MAX = 3.4028234663852886e38
ROUND = {torch.float32: (U32, 2.0 ** -149), torch.bfloat16: (2.0 ** -8, 2.0 ** -134),
         torch.float16: (2.0 ** -11, 2.0 ** -25)}
ROWS, TOP = 6, 5
# (type, mask): float16 holds its own lowest value only
MASKS = [(t, m) for t in (torch.float32, torch.bfloat16)
         for m in (torch.finfo(t).min, -1e9, -1e10, -1e30)] + \
    [(torch.float16, torch.finfo(torch.float16).min)]


def inputs(vocab, dtype, teacher, seed):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn((ROWS, vocab), generator=g) * 3).to(dtype)
    # entries among the first columns, so that later segments hold none
    index = torch.rand((ROWS, min(vocab, 200)), generator=g).topk(TOP, dim=1).indices
    values = torch.rand((ROWS, TOP), generator=g) * 6
    if teacher == "log_probs":
        mass = 0.3 + 0.4 * torch.rand((ROWS, 1), generator=g)
        values = torch.log_softmax(values, 1) + torch.log(mass)
    return logits, values, index


def span(z):
    """The range of the exponents that still count."""
    below = z.max() - z
    return float(below[below < 110].max())


def definition(logits, values, index, temp, teacher):
    """Loss and gradient of each row in float64, and the bounds of their
    float32 evaluation."""
    out = []
    for s, v, i in zip(logits.double(), values.double(), index):
        z = s / temp
        log_q = torch.log_softmax(z, 0)
        log_p = torch.log_softmax(v / temp, 0) if teacher == "logits" else v
        p = log_p.exp()
        terms = torch.where(p > 0, p * (log_p - log_q[i]), torch.zeros(()).double())
        scale = torch.where(p > 0, p * (log_p.abs() + log_q[i].abs()), torch.zeros(()).double())
        loss, scale = terms.sum(), scale.sum() + 1
        grad = torch.zeros_like(z).index_add_(0, i, -p)
        size = torch.zeros_like(z).index_add_(0, i, p)
        total, wide = p.sum(), span(z)
        if teacher == "log_probs":
            named = torch.zeros(len(z), dtype=torch.bool)
            named[i] = True
            r = 1.0 - float(total)
            log_rest = torch.logsumexp(log_q[~named], 0)
            share = torch.softmax(z.masked_fill(named, -math.inf), 0)
            loss = loss + r * (math.log(r) - log_rest)
            scale = scale + (r + 8) * abs(math.log(r)) + (r + 8 * U32) * log_rest.abs()
            grad = grad - r * share
            size = size + (r + 8) * share
            total = total + r
            wide = max(wide, span(z[~named]))
        if teacher == "logits":
            wide = max(wide, span(v / temp))
        c = 64 + 4 * wide + len(z) / 32
        out.append((temp * temp * loss, temp * (grad + total * log_q.exp()),
                    temp * temp * U32 * c * scale, temp * U32 * c * (size + total * log_q.exp())))
    return [torch.stack(t) for t in zip(*out)]


def check(logits, values, index, temp, teacher):
    dtype = logits.dtype
    loss, grad, loss_tol, grad_tol = definition(logits, values, index, temp, teacher)
    logits, values, index = logits.to(DEV), values.to(DEV), index.to(DEV)
    leaf = logits.detach().requires_grad_(True)
    each = distillation_loss(leaf, values, index, temperature=temp, teacher=teacher,
                             reduction="none")
    (g,) = torch.autograd.grad(each, leaf, torch.ones_like(each))
    _, both = distillation_value_and_grad(logits, values, index, temperature=temp,
                                          teacher=teacher, reduction="sum")
    got = each.detach().double().cpu()
    held = loss.abs() + loss_tol < F32_MAX  # else it may round to infinity
    assert not bool(got.isnan().any()) and bool(got[held].isfinite().all()), got
    over = (got - loss).abs() - (1.02 * loss_tol + U32 * loss.abs())
    assert bool((over[held] <= 0).all()), (float(over[held].max()), got, loss)
    assert bool((got[~held] >= F32_MAX / 2).all())
    r, sub = ROUND[dtype]
    for t in (g, both):
        over = (t.double().cpu() - grad).abs() - (1.02 * grad_tol + r * grad.abs() + sub)
        assert bool((over <= 0).all()), float(over.max())


# 30, 300: one launch; 20 001: three segments of 16-bit elements, five of float32
@pytest.mark.parametrize("temp", (0.5, 1.0, 2.0))
@pytest.mark.parametrize("dtype, mask", MASKS, ids=str)
@pytest.mark.parametrize("teacher", ("logits", "log_probs"))
@pytest.mark.parametrize("vocab", (30, 300, 2048, 20001))
def test_masked_stretches_rests_and_rows(vocab, teacher, dtype, mask, temp):
    logits, values, index = inputs(vocab, dtype, teacher, vocab)
    named = torch.zeros(logits.shape, dtype=torch.bool).scatter_(1, index, True)
    stretch = ~named & (torch.arange(vocab) >= vocab // 4)
    for where in (stretch, ~named, torch.ones_like(named)):
        check(torch.where(where, torch.tensor(mask, dtype=dtype), logits), values, index, temp,
              teacher)


@pytest.mark.parametrize("temp", (0.5, 1.0, 2.0))
@pytest.mark.parametrize("dtype, mask", MASKS, ids=str)
@pytest.mark.parametrize("teacher", ("logits", "log_probs"))
@pytest.mark.parametrize("vocab", (30, 20001))
def test_a_named_column_that_is_masked(vocab, teacher, dtype, mask, temp):
    logits, values, index = inputs(vocab, dtype, teacher, vocab + 1)
    logits.scatter_(1, index[:, 1:2], torch.tensor(mask, dtype=dtype).expand(ROWS, 1))
    check(logits, values, index, temp, teacher)


@pytest.mark.parametrize("temp", (0.5, 1.0, 2.0))
@pytest.mark.parametrize("mask", (torch.finfo(torch.float32).min, -1e9, -1e10, -1e30))
@pytest.mark.parametrize("vocab", (30, 20001))
def test_a_teacher_that_masks(vocab, mask, temp):
    """Some of a row's entries at the mask: no part of its softmax.  All of
    them: equal parts."""
    logits, values, index = inputs(vocab, torch.float32, "logits", vocab + 2)
    values[:3, 2:4] = mask
    values[3:] = mask
    check(logits, values, index, temp, "logits")
