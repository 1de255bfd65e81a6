"""Layer norm over rendered features (``gsx_layer_norm_fwd`` / ``gsx_layer_norm_bwd``).

Composited features are dimmed by the pixel's alpha; the norm takes that out of a
row before a decoder sees it.  No counterpart in the reference.
"""

from __future__ import annotations

import torch

from .. import _lib

__all__ = ["LayerNorm", "layer_norm"]


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        rows, stride = _lib.rows_of(x)
        w = None if weight is None else weight.contiguous()
        b = None if bias is None else bias.contiguous()
        y = _lib.contiguous_like(x)
        ctx.head = head = (_lib.DTYPES[x.dtype], rows.shape[0], rows.shape[1])
        _lib.launch("gsx_layer_norm_fwd", "layer_norm_fwd", x.device, *head, rows.data_ptr(), stride,
                    _lib.ptr(w), _lib.ptr(b), eps, y.data_ptr())
        ctx.save_for_backward(x, weight)
        ctx.eps = eps
        return y

    @staticmethod
    @_lib.once_differentiable("layer_norm")
    def backward(ctx, saved, g_y):
        x, weight = saved
        head, device = ctx.head, x.device
        rows, stride = _lib.rows_of(x)
        g_rows, g_stride = _lib.rows_of(g_y)
        w = None if weight is None else weight.contiguous()
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        g_x = _lib.contiguous_like(x) if need_x else None
        g_w = torch.empty(head[2], dtype=x.dtype, device=device) if need_w else None
        g_b = torch.empty(head[2], dtype=x.dtype, device=device) if need_b else None
        n = _lib.workspace_bytes("gsx_layer_norm_bwd_workspace_bytes", *head)
        ws = _lib.scratch(n, device) if need_w or need_b else None
        _lib.launch("gsx_layer_norm_bwd", "layer_norm_bwd", device, *head, rows.data_ptr(), stride,
                    _lib.ptr(w), g_rows.data_ptr(), g_stride, ctx.eps, _lib.ptr(g_x), _lib.ptr(g_w),
                    _lib.ptr(g_b), _lib.ptr(ws), n)
        return g_x, g_w, g_b, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None,
               bias: torch.Tensor | None = None, eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension of ``x``
    (..., C), with ``weight`` and ``bias`` (C,) or None (1 and 0); all of one type
    (float32, bfloat16, float16); differentiable with respect to all three, once (its
    gradient has none and says so).

    Statistics and sums are float32, the variance is that of the differences to the
    mean; outputs are rounded once.  A row with an infinite or NaN input comes out NaN,
    and no other row does."""
    if x.ndim < 1 or x.dtype not in _lib.DTYPES:
        raise ValueError("x must be (..., C) in float32, bfloat16 or float16.")
    if x.shape[-1] < 1:
        raise ValueError("x must have at least 1 column.")
    for t in (weight, bias):
        if t is not None and (t.dtype != x.dtype or t.shape != x.shape[-1:]):
            raise ValueError("weight and bias must have shape (C,) and x's type.")
    eps = float(eps)
    if not 1.2e-38 <= eps <= 3.0e38:
        raise ValueError("eps must be positive, finite and normal in float32 (from 1.2e-38 on).")
    _lib.require_device(x, weight, bias)
    return _LayerNorm.apply(x, weight, bias, eps)


class LayerNorm:
    """The norm with its weights: ``norm(x)`` normalises (..., C) rows.

    ``params`` are the leaf tensors ``weight`` (ones) and ``bias`` (zeros), as
    :class:`mlx3d_amd.optim.Adam` takes them."""

    def __init__(self, width: int, eps: float = 1e-5, dtype: torch.dtype = torch.float32,
                 device="cuda"):
        if width < 1:
            raise ValueError("x must have at least 1 column.")
        self.eps = float(eps)
        self.params = {"weight": torch.ones((width,), dtype=dtype, device=device),
                       "bias": torch.zeros((width,), dtype=dtype, device=device)}
        for p in self.params.values():
            p.requires_grad_(True)

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        return layer_norm(x, self.params["weight"], self.params["bias"], self.eps)
