"""The layer norm's gradient in a workspace of exactly the bytes asked for: nothing behind it
is written, and the gradients are those of the formulas."""

import pytest
import torch

from mlx3d_amd import _lib

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = 2.0 ** -24
TYPES = (torch.float32, torch.bfloat16, torch.float16)
# one element a lane, each size of team with one, two and three or four pieces a lane, rows
# that are read again; as many rows as give the most workgroups, where that is cheap
SIZES = [(270_000, 1), (270_000, 3), (140_000, 5), (70_000, 7), (200_000, 8), (100_000, 16),
         (60_000, 32), (50_000, 48), (30_000, 65), (20_000, 130), (10_000, 190), (9000, 300),
         (5000, 700), (3000, 1000), (2100, 1500), (1100, 1537), (700, 2050), (600, 4100),
         (600, 6000), (520, 8192), (300, 8193), (257, 20_001), (1, 64), (1, 8193), (0, 40)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_a_workspace_of_the_bytes_asked_for(size, dtype):
    """dw and db by chains of at most `rows` float32 additions; h itself is within a few
    hundred steps (a chain over the row's columns in the mean, the variance and the root)."""
    rows, width = size
    g = torch.Generator(device=DEV).manual_seed(rows + width)
    x, dy = (torch.randn(size, generator=g, device=DEV).to(dtype) for _ in range(2))
    w = torch.randn((width,), generator=g, device=DEV).to(dtype)
    L, kind = _lib.load(), _lib.DTYPES[dtype]
    need = L.gsx_layer_norm_bwd_workspace_bytes(kind, rows, width)
    room = torch.full((need + 4096,), 0xA5, dtype=torch.uint8, device=DEV)
    dw, db = (torch.empty((width,), dtype=dtype, device=DEV) for _ in range(2))
    dx = torch.empty_like(x)
    _lib.check(L.gsx_layer_norm_bwd(
        kind, rows, width, x.data_ptr() or None, width, w.data_ptr(), dy.data_ptr() or None, width,
        1e-5, dx.data_ptr() or None, dw.data_ptr(), db.data_ptr(), room.data_ptr(), need,
        _lib.stream_handle(torch.device(DEV))), "gsx_layer_norm_bwd")
    assert bool((room[need:] == 0xA5).all())
    x, dy = x.double(), dy.double()
    d = x - x.mean(dim=1, keepdim=True)
    h = d / ((d * d).mean(dim=1, keepdim=True) + 1e-5).sqrt()
    step = torch.finfo(dtype).eps / 2
    for got, terms, each in ((dw, dy * h, 64 + width), (db, dy, 0)):
        want, size_ = terms.sum(dim=0), terms.abs().sum(dim=0)
        if each:  # h's own error, absolute in rows of few columns: |x| / spread times steps
            size_ = size_ + dy.abs().sum(dim=0)
        bound = (rows + 1 + each) * U * size_ + step * want.abs() + 2.0 ** -25
        assert bool(((got.double() - want).abs() <= bound).all())
