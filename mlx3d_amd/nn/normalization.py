"""Layer norm over rendered features (``gsx_layer_norm_fwd`` / ``gsx_layer_norm_bwd``).

Composited features are dimmed by the pixel's alpha; the norm takes that out of a
row before a decoder sees it.  No counterpart in the reference.
"""

from __future__ import annotations

import torch

from .. import _lib
from ..profiling import stage

__all__ = ["LayerNorm", "layer_norm"]


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        rows, stride = _lib.rows_of(x)
        w, b = (None if t is None else t.contiguous() for t in (weight, bias))
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        head = (_lib.DTYPES[x.dtype], rows.shape[0], x.shape[-1])
        with _lib.on_device(x.device), stage("layer_norm_fwd"):
            _lib.check(_lib.load().gsx_layer_norm_fwd(
                *head, _lib.ptr(rows), stride, _lib.ptr(w), _lib.ptr(b), eps, _lib.ptr(y),
                _lib.stream_handle(x.device)), "gsx_layer_norm_fwd")
        ctx.save_for_backward(x, weight)
        ctx.head, ctx.eps = head, eps
        return y

    @staticmethod
    @_lib.once_differentiable("layer_norm")
    def backward(ctx, saved, g_y):
        x, weight = saved
        L = _lib.load()
        rows, stride = _lib.rows_of(x)
        g_rows, g_stride = _lib.rows_of(g_y)
        w = None if weight is None else weight.contiguous()
        need = ctx.needs_input_grad
        g_x = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need[0] else None
        g_w, g_b = (torch.empty(x.shape[-1:], dtype=x.dtype, device=x.device) if k else None
                    for k in need[1:3])
        n = _lib.check(int(L.gsx_layer_norm_bwd_workspace_bytes(*ctx.head)),
                       "gsx_layer_norm_bwd_workspace_bytes")
        ws = torch.empty((n,), dtype=torch.uint8, device=x.device)
        with _lib.on_device(x.device), stage("layer_norm_bwd"):
            _lib.check(L.gsx_layer_norm_bwd(
                *ctx.head, _lib.ptr(rows), stride, _lib.ptr(w), _lib.ptr(g_rows), g_stride,
                ctx.eps, _lib.ptr(g_x), _lib.ptr(g_w), _lib.ptr(g_b), _lib.ptr(ws), n,
                _lib.stream_handle(x.device)), "gsx_layer_norm_bwd")
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
