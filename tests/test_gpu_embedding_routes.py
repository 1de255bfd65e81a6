"""The table's gradient on every route of its sort, its tiles and their joins.

Incoming gradients are small whole numbers, so every partial sum is a whole number below
2^24, which float32 holds: whatever the order, the gradient is the exact sum, rounded once
to the table's type.  There is no tolerance."""

import pytest
import torch

from mlx3d_amd.nn import embedding

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = (torch.float32, torch.bfloat16, torch.float16)
CHUNK = 4096  # tokens that a workgroup of the sort holds; above 4 of them there are several


def numbers(shape, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randint(-7, 8, shape, generator=g, device=DEV, dtype=torch.int8).to(dtype)


def gradient(k, rows, dy):
    table = torch.zeros((rows, dy.shape[1]), dtype=dy.dtype, device=DEV, requires_grad=True)
    return torch.autograd.grad(embedding(k, table), table, dy)[0]


def sums(k, rows, dy):
    """By row, exact: differences of running sums over the sorted tokens."""
    k, order = torch.sort(k)
    ends = torch.searchsorted(k, torch.arange(rows + 1, device=DEV))
    run = torch.zeros((len(k) + 1, dy.shape[1]), dtype=torch.float64, device=DEV)
    run[1:] = dy[order].double().T.contiguous().cumsum(dim=1).T
    return run[ends[1:]] - run[ends[:-1]]


def check(k, rows, dy):
    got = gradient(k, rows, dy)
    there = (k >= 0) & (k < rows)
    own, told = k[there].long(), dy[there]
    # what the docstring says; 7 is the largest
    assert 7 * len(own) < 2 ** 24 or float(sums(own, rows, told.abs()).max()) < 2 ** 24
    assert torch.equal(got, sums(own, rows, told).to(dy.dtype))


def some_of(count, rows, live, seed):
    """`live` of `count` indices name a row, the others lie on either side of the table."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    k = torch.randint(0, rows, (count,), generator=g, device=DEV)
    gone = torch.randperm(count, generator=g, device=DEV)[live:]
    k[gone] = torch.where(gone % 3 == 0, rows + gone, -1 - gone)
    return k


# -- the sort: passes by the rows' bits, tokens that name no row --

# one pass of 8 bits, of 12; two of 8; two of 12; three of 12, on both sides of each change
ROWS = (2, 255, 256, 257, 4096, 4097, 5000, 65_536, 65_537, 1 << 24, (1 << 24) + 1)
# all; none; one; short of a chunk, a chunk and a token more, as many as end a chunk later
LIVE = (5 * CHUNK + 77, 0, 1, CHUNK - 1, CHUNK, CHUNK + 1, 3 * CHUNK, 3 * CHUNK + 5)


@pytest.mark.parametrize("live", LIVE)
@pytest.mark.parametrize("rows", ROWS)
def test_passes(rows, live):
    count = 5 * CHUNK + 77
    k = some_of(count, rows, live, seed=rows + live)
    assert int(((k >= 0) & (k < rows)).sum()) == live
    check(k.int() if live % 2 else k, rows, numbers((count, 3), torch.float32, seed=live))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows", ROWS)
def test_passes_over_many_chunks(rows, dtype):
    """Prefixes over more chunks than a thread keeps in registers (16 stretches of 16)."""
    count = 300 * CHUNK - 3
    k = some_of(count, rows, count - count // 7, seed=rows)
    check(k, rows, numbers((count, 1), dtype, seed=rows))


@pytest.mark.parametrize("rows", (256, 300, 5000, 70_000, (1 << 24) + 1))
def test_passes_are_stable(rows):
    """Tokens of a row stay in their order, on which the rounding of sums depends: the
    gradient has the bits that the same tokens, sorted beforehand, give."""
    count = 7 * CHUNK + 9
    g = torch.Generator(device=DEV).manual_seed(1)
    named = torch.randperm(rows, generator=g, device=DEV)[:200]
    k = named[torch.randint(0, 200, (count,), generator=g, device=DEV)]
    dy = torch.randn((count, 3), generator=g, device=DEV)
    order = torch.sort(k, stable=True).indices
    first = gradient(k, rows, dy)
    assert torch.equal(first, gradient(k[order], rows, dy[order]))
    assert torch.equal(first, gradient(k, rows, dy))


def test_the_last_rows_of_a_long_table():
    """Digits of 0 and of all ones in every pass."""
    for rows in (4097, 65_536, 65_537, 1 << 24, (1 << 24) + 1):
        count = 5 * CHUNK
        k = torch.tensor([0, rows - 1, rows // 2, 255, 256, 4095, 4096], device=DEV)
        k = k.repeat(count // 7 + 1)[:count]
        check(k, rows, numbers((count, 2), torch.float32, seed=rows))


# -- where the number of tokens changes what runs --

@pytest.mark.parametrize("how", ("one", "turns", "few", "gone"))
@pytest.mark.parametrize("count", (7, 8, 9, 63, 64, 65, 1023, 1024, 1025, CHUNK - 1, CHUNK,
                                   CHUNK + 1, 4 * CHUNK - 1, 4 * CHUNK, 4 * CHUNK + 1))
def test_counts(count, how):
    rows = 300
    g = torch.Generator(device=DEV).manual_seed(count)
    k = {"one": torch.full((count,), 299, device=DEV),
         "turns": torch.arange(count, device=DEV) % rows,
         "few": (rows * torch.rand((count,), generator=g, device=DEV) ** 6).long(),
         "gone": torch.where(torch.rand((count,), generator=g, device=DEV) < 0.9, -1, 5)}[how]
    for width, dtype in ((9, torch.bfloat16), (33, torch.float32)):
        check(k, rows, numbers((count, width), dtype, seed=count))


# -- tiles and joins: every team of lanes, rows over any number of blocks --

def pieces_of(width, dtype):
    vec = 16 // dtype.itemsize
    return width if width < vec else -(-width // vec)


def block_of(count, width, dtype):
    """Sorted tokens of a workgroup's tiles, as the kernels take them: tiles of 256 down to
    8 while there are fewer than 2^16 lanes, times the teams of 256 threads."""
    pieces, tile, lanes = pieces_of(width, dtype), 256, 1
    while tile > 8 and count * pieces < tile << 16:
        tile //= 2
    while lanes < 64 and lanes < pieces:
        lanes *= 2
    return tile * (256 // lanes), tile


def shuffled(lengths, seed):
    """Indices with lengths[v] tokens of row v, in a random order."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    n = torch.tensor(lengths, device=DEV)
    k = torch.repeat_interleave(torch.arange(len(lengths), device=DEV), n)
    return k[torch.randperm(len(k), generator=g, device=DEV)]


# element by element and in pieces, each number of lanes, and rows of more than 64 pieces
WIDTHS = {torch.float32: (1, 2, 3, 4, 7, 13, 27, 50, 100, 255, 520),
          torch.bfloat16: (1, 2, 4, 7, 8, 15, 27, 50, 100, 200, 511, 1030)}
WIDTHS[torch.float16] = WIDTHS[torch.bfloat16]
TEAMS = [(t, w) for t in TYPES for w in WIDTHS[t]]


@pytest.mark.parametrize("dtype, width", TEAMS, ids=str)
def test_rows_over_many_blocks(dtype, width):
    """Rows over 31, 32 (joined by a team), 33, 34 and 300 blocks (joined by a workgroup, up
    to eight lanes a row several of them in its range), from the middle of a block to the
    middle of another, next to rows of no token, of one, and of a block."""
    block, tile = block_of(0, width, dtype)
    lengths = [block // 2, 0, 1]
    for span in (31, 1, 32, 33, 2, 34, 0, 300 if pieces_of(width, dtype) <= 64 else 40):
        lengths += [span * block, 1]
    lengths.append(block + 3)
    count = sum(lengths)
    assert block_of(count, width, dtype) == (block, tile)
    check(shuffled(lengths, seed=width), len(lengths), numbers((count, width), dtype, width))


@pytest.mark.parametrize("dtype, width", TEAMS, ids=str)
def test_rows_on_the_borders_of_blocks(dtype, width):
    """Rows that begin or end where a tile or a block does, or a token beside it; tokens of a
    last block that is full, or holds one."""
    block, tile = block_of(0, width, dtype)
    lengths = [block, tile, tile - 1, 1, block - 2 * tile, 2 * block, block - 1, 1, 1, block + 1,
               40 * block - 2, tile + 1, block - tile - 1, block]
    for tail in ([], [1], [block - 1, 1]):
        counts = lengths + tail
        assert block_of(sum(counts), width, dtype) == (block, tile)
        check(shuffled(counts, seed=width), len(counts) + 2,
              numbers((sum(counts), width), dtype, width))


@pytest.mark.parametrize("dtype, width", [(torch.float32, 4), (torch.float32, 50),
                                          (torch.bfloat16, 27), (torch.float16, 7)], ids=str)
def test_one_block_and_two(dtype, width):
    """Where the join's launch begins."""
    block, _ = block_of(0, width, dtype)
    for count in (block - 1, block, block + 1, 2 * block, 2 * block + 1):
        for rows in (1, 3, count):
            check(torch.arange(count, device=DEV) * 7 % rows, rows,
                  numbers((count, width), dtype, count))


@pytest.mark.parametrize("size, tile", [((1_100_003, 64), 256), ((700_001, 64), 128),
                                        ((600_001, 32), 64), ((300_000, 32), 32),
                                        ((300_000, 16), 16)], ids=str)
def test_larger_tiles(size, tile):
    count, width = size
    assert block_of(count, width, torch.float32)[1] == tile
    g = torch.Generator(device=DEV).manual_seed(tile)
    for k in ((5000 * torch.rand((count,), generator=g, device=DEV) ** 4).long(),
              torch.arange(count, device=DEV) % 4999):
        check(k, 5000, numbers(size, torch.float32, seed=tile))
