"""Dropout whose mask is never stored (``gsx_dropout``).

Which elements are kept follows from a seed, a counter and the element's place, so
the gradient forms the mask again.  No counterpart in the reference.
"""

from __future__ import annotations

import torch

from .. import _lib

__all__ = ["Dropout", "dropout"]


def dropout(x: torch.Tensor, p: float, seed: int, offset: int | torch.Tensor = 0,
            residual: torch.Tensor | None = None) -> torch.Tensor:
    """Each element of ``x`` with probability 1 - ``p`` divided by 1 - p, else 0; with a
    ``residual`` of x's shape and type, that plus the residual, rounded once.  float32,
    bfloat16 or float16; differentiable with respect to both, once (its gradient has none
    and says so).

    Which elements are kept follows from ``seed`` (0 to 2^64 - 1), ``offset`` (0 to
    2^63 - 1) and the element's place in row-major order alone: the generator is
    Philox4x32-10 (include/gsx.h has the counters).  A training step takes a seed for
    each place where it drops, and its step as the offset: a number, or a one-element
    int64 tensor on the device, which a captured graph reads at every replay (non-negative;
    move it on after the gradient, not before).

    What is dropped counts as 0 whatever it holds; p = 1 drops everything."""
    if x.dtype not in _lib.DTYPES:
        raise ValueError("x must be float32, bfloat16 or float16.")
    if residual is not None and (residual.dtype != x.dtype or residual.shape != x.shape):
        raise ValueError("the residual must have x's shape and type.")
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError("p must lie in [0, 1].")
    if not isinstance(seed, int) or not 0 <= seed < 1 << 64:
        raise ValueError("seed must be a whole number from 0 to 2^64 - 1.")
    if isinstance(offset, torch.Tensor):
        if offset.dtype != torch.int64 or offset.numel() != 1:
            raise ValueError("an offset on the device must be one int64.")
        offset, at = 0, offset
    else:
        if not isinstance(offset, int) or not 0 <= offset < 1 << 63:
            raise ValueError("offset must be a whole number from 0 to 2^63 - 1.")
        at = None
    _lib.require_device(x, residual, at)
    return _lib.autograd().dropout(x, residual, p, seed, offset, at)


class Dropout:
    """Dropout at one place of a network: ``drop(x, residual)`` in a training step,
    ``drop.advance()`` after its gradient, so that the next step draws another mask.

    The step is counted on the device (``step``), so both may be captured into a graph.
    While ``training`` is False, x (plus the residual) comes back undropped."""

    def __init__(self, p: float, seed: int, device="cuda"):
        if not 0.0 <= float(p) <= 1.0:
            raise ValueError("p must lie in [0, 1].")
        if not isinstance(seed, int) or not 0 <= seed < 1 << 64:
            raise ValueError("seed must be a whole number from 0 to 2^64 - 1.")
        self.p, self.seed, self.training = float(p), seed, True
        self.step = torch.zeros((1,), dtype=torch.int64, device=device)

    def __call__(self, x: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
        if not self.training:
            return x if residual is None else x + residual
        return dropout(x, self.p, self.seed, self.step, residual)

    def advance(self) -> None:
        self.step += 1
