"""Layer norm over rendered features (``gsx_layer_norm_fwd`` / ``gsx_layer_norm_bwd``).

Composited features are dimmed by the pixel's alpha; the norm takes that out of a
row before a decoder sees it.  No counterpart in the reference.
"""

from __future__ import annotations

import torch

from .. import _lib

__all__ = ["LayerNorm", "layer_norm"]


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None,
               bias: torch.Tensor | None = None, eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension of ``x``
    (..., C), with ``weight`` and ``bias`` (C,) or None (1 and 0); all of one type
    (float32, bfloat16, float16); differentiable with respect to all three, once (its
    gradient has none and says so).

    Statistics and sums are float32, the variance is that of the differences to the
    mean; outputs are rounded once.  A row with an infinite or NaN input, or whose float32
    sum overflows, comes out NaN, and no other row does; one whose float32 variance
    alone overflows (differences from about 1e19) is normalised to zeros.  At most 2^20
    columns and 2^30 rows; more is refused (``GsxError``)."""
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
    return _lib.autograd().layer_norm(x, weight, bias, eps)


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
