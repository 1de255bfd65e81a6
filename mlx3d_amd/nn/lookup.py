"""Rows of a table by their indices (``gsx_embed_fwd`` / ``gsx_embed_bwd``).

Gaussians that share a codebook, pixels that take their view's appearance, tokens
of a text: each names a row of a table, and the table's gradient is the sum over
those that named a row.  No counterpart in the reference.
"""

from __future__ import annotations

import torch

from .. import _lib

__all__ = ["Embedding", "embedding"]


def embedding(indices: torch.Tensor, table: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """(..., C) = ``scale`` times the rows of ``table`` (V, C) that ``indices``
    (..., int32 or int64) name; zeros where an index lies outside [0, V), so -1 stands
    for no row.  ``table`` is float32, bfloat16 or float16; differentiable with respect
    to it, once (its gradient has none and says so).

    The gradient is dense, summed in float32 in an order that the indices fix, so the
    same inputs give the same bits.  Rows that no index names have zeros.  At most 2^30
    indices and rows and 2^20 columns; more is refused (``GsxError``)."""
    if indices.dtype not in (torch.int32, torch.int64):
        raise ValueError("indices must be int32 or int64.")
    if table.ndim != 2 or table.dtype not in _lib.DTYPES:
        raise ValueError("table must be (V, C) in float32, bfloat16 or float16.")
    if min(table.shape) < 1:
        raise ValueError("the table must have at least 1 row and 1 column.")
    scale = float(scale)
    if not abs(scale) < 3.4e38:
        raise ValueError("scale must be finite in float32.")
    _lib.require_device(indices, table)
    return _lib.autograd().embedding(indices, table, scale)


class Embedding:
    """A table with its scale: ``table(indices)`` looks rows up.

    ``params`` holds the leaf tensor ``table`` (normal with variance 1 / scale^2, so
    that what is looked up has variance 1), as :class:`mlx3d_amd.optim.Adam` takes it."""

    def __init__(self, rows: int, width: int, scale: float = 1.0,
                 dtype: torch.dtype = torch.float32, device="cuda", seed: int = 0):
        if min(rows, width) < 1:
            raise ValueError("the table must have at least 1 row and 1 column.")
        if not 0.0 < abs(float(scale)) < 3.4e38:
            raise ValueError("scale must be finite in float32, and not 0.")
        self.scale = float(scale)
        g = torch.Generator().manual_seed(seed)
        table = torch.randn((rows, width), generator=g) / self.scale
        self.params = {"table": table.to(device=device, dtype=dtype).requires_grad_(True)}

    def __call__(self, indices: torch.Tensor) -> torch.Tensor:
        return embedding(indices, self.params["table"], self.scale)
