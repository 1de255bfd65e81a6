"""Rows of a table by their indices (``gsx_embed_fwd`` / ``gsx_embed_bwd``).

Gaussians that share a codebook, pixels that take their view's appearance, tokens
of a text: each names a row of a table, and the table's gradient is the sum over
those that named a row.  No counterpart in the reference.
"""

from __future__ import annotations

import torch

from .. import _lib

__all__ = ["Embedding", "embedding"]


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, indices, table, scale):
        held = indices.contiguous()
        rows, stride = _lib.rows_of(table)
        count, device = held.numel(), table.device
        y = torch.empty((*held.shape, table.shape[1]), dtype=table.dtype, device=device)
        ctx.head = head = (_lib.DTYPES[table.dtype], count, *table.shape)
        ctx.how = how = (int(indices.dtype == torch.int64), scale)
        _lib.launch("gsx_embed_fwd", "embed_fwd", device, *head, held.data_ptr(), how[0],
                    rows.data_ptr(), stride, scale, y.data_ptr())
        ctx.save_for_backward(indices)
        return y

    @staticmethod
    @_lib.once_differentiable("embedding")
    def backward(ctx, saved, g_y):
        held = saved[0].contiguous()
        head, (index64, scale), device = ctx.head, ctx.how, g_y.device
        rows, stride = _lib.rows_of(g_y)
        g_table = torch.empty(head[2:], dtype=g_y.dtype, device=device)
        n = _lib.workspace_bytes("gsx_embed_bwd_workspace_bytes", *head)
        ws = _lib.scratch(n, device)
        _lib.launch("gsx_embed_bwd", "embed_bwd", device, *head, held.data_ptr(), index64,
                    rows.data_ptr(), stride, scale, g_table.data_ptr(), ws.data_ptr(), n)
        return None, g_table, None


def embedding(indices: torch.Tensor, table: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """(..., C) = ``scale`` times the rows of ``table`` (V, C) that ``indices``
    (..., int32 or int64) name; zeros where an index lies outside [0, V), so -1 stands
    for no row.  ``table`` is float32, bfloat16 or float16; differentiable with respect
    to it, once (its gradient has none and says so).

    The gradient is dense, summed in float32 in an order that the indices fix, so the
    same inputs give the same bits.  Rows that no index names have zeros."""
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
    return _Embedding.apply(indices, table, scale)


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
