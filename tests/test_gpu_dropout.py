"""Dropout against the generator's definition in NumPy, its values against 64 bits, and
what a training loop does with it."""

import numpy as np
import pytest
import torch

from mlx3d_amd.nn import Dropout, dropout

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = (torch.float32, torch.bfloat16, torch.float16)
ROUND = {torch.float32: (2.0 ** -24, 2.0 ** -150), torch.bfloat16: (2.0 ** -8, 2.0 ** -134),
         torch.float16: (2.0 ** -11, 2.0 ** -25)}


def philox(counter, key):
    """Philox4x32 with ten rounds, in 64-bit integers: (n, 4) words of (n, 4) counters."""
    c = counter.astype(np.uint64)
    k0, k1 = np.uint64(key & 0xFFFFFFFF), np.uint64(key >> 32)
    low = np.uint64(0xFFFFFFFF)
    for _ in range(10):
        p, q = c[:, 0] * np.uint64(0xD2511F53), c[:, 2] * np.uint64(0xCD9E8D57)
        c = np.stack([(q >> np.uint64(32)) ^ c[:, 1] ^ k0, q & low,
                      (p >> np.uint64(32)) ^ c[:, 3] ^ k1, p & low], axis=1)
        k0, k1 = (k0 + np.uint64(0x9E3779B9)) & low, (k1 + np.uint64(0xBB67AE85)) & low
    return c.astype(np.uint32)


def test_the_generator_itself():
    """The known answers that its authors publish with it."""
    full = 0xFFFFFFFF
    for counter, key, words in (
            ((0, 0, 0, 0), 0, (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
            ((full,) * 4, 2 ** 64 - 1, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
            ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), 0x299F31D0A4093822,
             (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))):
        assert philox(np.array([counter], dtype=np.uint64), key)[0].tolist() == list(words)


def numbers(first, count, seed, offset):
    """The 32-bit numbers of elements first .. first + count - 1."""
    element = np.arange(first, first + count, dtype=np.uint64)
    block = element // np.uint64(8)
    half = []
    for stream in (0, 1 << 63):
        b = block + np.uint64(stream)
        counter = np.stack([b & np.uint64(0xFFFFFFFF), b >> np.uint64(32),
                            np.full_like(b, offset & 0xFFFFFFFF), np.full_like(b, offset >> 32)], 1)
        words = philox(counter, seed)
        word = words[np.arange(count), (element % np.uint64(8)).astype(int) // 2]
        half.append((word >> (16 * (element % np.uint64(2))).astype(np.uint32)) & np.uint32(0xFFFF))
    return half[0].astype(np.uint64) << np.uint64(16) | half[1].astype(np.uint64)


def mask(shape, p, seed, offset):
    n = int(np.prod(shape))
    kept = numbers(0, n, seed, offset) >= np.uint64(round(p * 2 ** 32))
    return torch.from_numpy(kept).view(shape).to(DEV)


def inputs(shape, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(shape, generator=g).to(dtype).to(DEV) for _ in range(3)]


def check(got, x, kept, p, residual=None):
    """One product and one sum in float32, and a rounding to the type."""
    ulp, sub = ROUND[x.dtype]
    term = torch.where(kept, x.double() / (1 - p), 0.0) if p < 1 else torch.zeros_like(x).double()
    want = term + (0.0 if residual is None else residual.double())
    bound = 2 * 2.0 ** -24 * (term.abs() + want.abs()) + ulp * want.abs() + sub
    assert got.dtype == x.dtype and got.shape == x.shape
    assert bool(((got.double() - want).abs() <= bound).all())
    if residual is None:
        assert bool((got[~kept] == 0).all())


# no block of eight, one, odd ends, both sides of a workgroup's 2048 elements
SHAPES = [(1,), (7,), (8,), (3, 3), (2047,), (2, 1024), (2049,), (64, 64), (33, 21), (5, 7, 11),
          (1000, 100)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_values_and_gradients(shape, dtype):
    p, seed, offset = 0.3, 0x123456789ABCDEF0 + len(shape), 5
    x, residual, dy = inputs(shape, dtype, seed=sum(shape))
    kept = mask(shape, p, seed, offset)
    for base in (None, residual):
        leaves = [t.detach().requires_grad_(True) for t in (x, base) if t is not None]
        y = dropout(leaves[0], p, seed, offset, *leaves[1:])
        check(y.detach(), x, kept, p, base)
        grads = torch.autograd.grad(y, leaves, dy)
        check(grads[0], dy, kept, p)
        if base is not None:
            assert torch.equal(grads[1], dy)


@pytest.mark.parametrize("p", (0.0, 2.0 ** -33, 2.0 ** -32, 1e-5, 0.1, 0.25, 0.5, 0.9, 1 - 2.0 ** -32,
                               1 - 2.0 ** -34, 1.0))
@pytest.mark.parametrize("seed, offset", ((0, 0), (2 ** 64 - 1, 2 ** 63 - 1), (1 << 40, 1 << 33)))
def test_every_probability(p, seed, offset):
    x, residual, _ = inputs((3001,), torch.float32)
    kept = mask((3001,), p, seed, offset)
    check(dropout(x, p, seed, offset), x, kept, p)
    if p == 0.0:
        assert torch.equal(dropout(x, p, seed, offset), x)
    if p >= 1 - 2.0 ** -34:
        assert not bool(dropout(x, p, seed, offset).any())
        assert torch.equal(dropout(x, p, seed, offset, residual), residual)


def test_lower_halves_decide():
    """Thresholds at an element's own number and one above it: where the upper half is
    the threshold's, the lower half tells."""
    seed, offset, n = 99, 3, 4096
    u = numbers(0, n, seed, offset)
    x = torch.ones((n,), device=DEV)
    for at in (0, 17, 2222, 4095):
        for threshold in (int(u[at]), int(u[at]) + 1):
            y = dropout(x, threshold / 2 ** 32, seed, offset)
            assert torch.equal(y != 0, torch.from_numpy(u >= np.uint64(threshold)).to(DEV))


def test_share_and_independence():
    """A million elements: the kept share within five deviations, and so is what two
    steps, two seeds and neighbouring elements have in common."""
    n, p = 1 << 20, 0.25
    x = torch.ones((n,), device=DEV)
    masks = [dropout(x, p, seed, step) != 0 for seed, step in ((1, 0), (1, 1), (2, 0))]
    masks.append(masks[0].roll(1))
    for i, m in enumerate(masks):
        assert abs(float(m.double().mean()) - 0.75) < 5 * (0.75 * 0.25 / n) ** 0.5
        for k in masks[:i]:
            both = 0.75 ** 2
            assert abs(float((m & k).double().mean()) - both) < 5 * (both * (1 - both) / n) ** 0.5


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_what_is_dropped_counts_as_zero(dtype):
    x = torch.full((4000,), float("nan"), dtype=dtype, device=DEV)
    x[1::2] = float("inf")
    kept = mask((4000,), 0.5, 4, 0)
    y = dropout(x, 0.5, 4)
    assert torch.equal(y == 0, ~kept)
    assert torch.equal(dropout(x, 0.5, 4, 0, torch.ones_like(x)) == 1, ~kept)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_layouts(dtype):
    """The mask goes by an element's place in row-major order, however it lies."""
    x, residual, dy = inputs((40, 37), dtype, seed=2)
    want = dropout(x, 0.4, 8, 2, residual)
    wide = torch.full((40, 50), float("nan"), dtype=dtype, device=DEV)
    wide[:, 5:42] = x
    odd = torch.full((40 * 37 + 1,), float("nan"), dtype=dtype, device=DEV)
    odd[1:] = residual.reshape(-1)
    assert torch.equal(dropout(wide[:, 5:42], 0.4, 8, 2, odd[1:].view(40, 37)), want)
    turned = x.t().contiguous().t().requires_grad_(True)
    y = dropout(turned, 0.4, 8, 2, residual.t().contiguous().t())
    assert torch.equal(y.detach(), want)
    (grad,) = torch.autograd.grad(y, turned, dy.t().contiguous().t())
    assert torch.equal(grad, dropout(dy, 0.4, 8, 2))
    odd_x = torch.full((40 * 37 + 3,), float("nan"), dtype=dtype, device=DEV)
    odd_x[3:] = x.reshape(-1)
    assert torch.equal(dropout(odd_x[3:].view(40, 37), 0.4, 8, 2, residual), want)
    assert torch.equal(dropout(x[:1].expand(3, 37), 0.4, 8),
                       dropout(x[:1].expand(3, 37).contiguous(), 0.4, 8))
    one = x[0, 0]
    assert dropout(one, 0.0, 1).shape == () and float(dropout(one, 0.0, 1)) == float(one)


def test_no_elements():
    x = torch.empty((0, 5), device=DEV, requires_grad=True)
    y = dropout(x, 0.5, 1)
    assert y.shape == (0, 5) and torch.autograd.grad(y.sum(), x)[0].shape == (0, 5)


def test_a_counter_on_the_device():
    x, residual, dy = inputs((500, 9), torch.float32)
    for step in (0, 1, 2 ** 31, 2 ** 33 + 5):
        at = torch.full((1,), step, dtype=torch.int64, device=DEV)
        leaf = x.detach().requires_grad_(True)
        y = dropout(leaf, 0.2, 3, at, residual)
        assert torch.equal(y.detach(), dropout(x, 0.2, 3, step, residual))
        (grad,) = torch.autograd.grad(y, leaf, dy)
        assert torch.equal(grad, dropout(dy, 0.2, 3, step))


def test_a_counter_that_moves_before_the_gradient_is_noticed():
    drop = Dropout(0.5, seed=1)
    x = torch.ones((100,), device=DEV, requires_grad=True)
    y = drop(x)
    drop.advance()
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()


def test_module():
    drop = Dropout(0.5, seed=7)
    x, residual, _ = inputs((64, 64), torch.float32)
    first = drop(x)
    assert torch.equal(first, drop(x)) and torch.equal(first, dropout(x, 0.5, 7, 0))
    drop.advance()
    assert torch.equal(drop(x, residual), dropout(x, 0.5, 7, 1, residual))
    drop.training = False
    assert torch.equal(drop(x), x) and torch.equal(drop(x, residual), x + residual)


def test_captured_steps_draw_new_masks():
    drop = Dropout(0.3, seed=21)
    x, residual, dy = inputs((200, 33), torch.float32)
    leaf = x.detach().requires_grad_(True)

    def step():
        y = drop(leaf, residual)
        (grad,) = torch.autograd.grad(y, leaf, dy)
        drop.advance()
        return y.detach(), grad

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    drop.step.zero_()
    for k in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], dropout(x, 0.3, 21, k, residual))
        assert torch.equal(got[1], dropout(dy, 0.3, 21, k))
        assert int(drop.step) == k + 1


def test_more_elements_than_32_bits_count():
    """The last elements of more than 2^32, against the generator's definition."""
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("takes 30 GB of device memory")
    n = (1 << 32) + 13
    x = torch.ones((n,), dtype=torch.bfloat16, device=DEV)
    y = dropout(x, 0.5, 5, 1)
    for first in ((1 << 31) - 100, (1 << 32) - 100, n - 100):
        kept = numbers(first, 100, 5, 1) >= np.uint64(1 << 31)
        assert torch.equal((y[first:first + 100] != 0).cpu(), torch.from_numpy(kept))
