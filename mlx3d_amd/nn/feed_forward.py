"""The gated feed-forward block that decodes rendered features
(``gsx_ffn_fwd`` / ``gsx_ffn_bwd``).

A scene's Gaussians carry a few feature channels that
``render_gaussian_features`` composites per pixel; this block takes each row
of them into a teacher's space (class logits, an embedding):

    y = (act(x w_gate^T) * (x w_up^T)) w_down^T

No counterpart in the reference, whose ``nn`` package holds NeRF networks.
"""

from __future__ import annotations

import math

import torch

from .. import _lib
from ..profiling import stage

__all__ = ["GatedFeedForward", "gated_feed_forward"]

_ACTIVATIONS = {"silu": 0, "gelu": 1, "sigmoid": 2}


class _GatedFeedForward(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, act):
        L = _lib.load()
        rows, stride = _lib.rows_of(x)
        weights = [w.contiguous() for w in (w_gate, w_up, w_down)]
        head = (_lib.DTYPES[x.dtype], act, rows.shape[0], x.shape[-1], w_gate.shape[0],
                w_down.shape[0])
        y = torch.empty((*x.shape[:-1], w_down.shape[0]), dtype=x.dtype, device=x.device)
        n = _lib.check(int(L.gsx_ffn_fwd_workspace_bytes(*head)), "gsx_ffn_fwd_workspace_bytes")
        ws = torch.empty((n,), dtype=torch.uint8, device=x.device) if n else None
        with stage("ffn_fwd"):
            _lib.check(L.gsx_ffn_fwd(*head, _lib.ptr(rows), stride, *map(_lib.ptr, weights),
                                     _lib.ptr(y), _lib.ptr(ws), n, _lib.stream_handle(x.device)),
                       "gsx_ffn_fwd")
        ctx.save_for_backward(x, w_gate, w_up, w_down)
        ctx.head = head
        return y

    @staticmethod
    @_lib.once_differentiable("gated_feed_forward")
    def backward(ctx, saved, g_y):
        x, *weights = saved
        L = _lib.load()
        rows, stride = _lib.rows_of(x)
        g_rows, g_stride = _lib.rows_of(g_y)
        held = [w.contiguous() for w in weights]
        need = ctx.needs_input_grad
        g_x = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need[0] else None
        pair = need[1] or need[2]
        g_gate, g_up = ((torch.empty(w.shape, dtype=w.dtype, device=w.device) for w in weights[:2])
                        if pair else (None, None))
        g_down = (torch.empty(weights[2].shape, dtype=x.dtype, device=x.device) if need[3]
                  else None)
        n = _lib.check(int(L.gsx_ffn_bwd_workspace_bytes(*ctx.head)),
                       "gsx_ffn_bwd_workspace_bytes")
        ws = torch.empty((n,), dtype=torch.uint8, device=x.device)
        with stage("ffn_bwd"):
            _lib.check(L.gsx_ffn_bwd(*ctx.head, _lib.ptr(rows), stride, *map(_lib.ptr, held),
                                     _lib.ptr(g_rows), g_stride, _lib.ptr(g_x), _lib.ptr(g_gate),
                                     _lib.ptr(g_up), _lib.ptr(g_down), _lib.ptr(ws), n,
                                     _lib.stream_handle(x.device)), "gsx_ffn_bwd")
        return g_x, g_gate if need[1] else None, g_up if need[2] else None, g_down, None


def gated_feed_forward(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor,
                       w_down: torch.Tensor, activation: str = "silu") -> torch.Tensor:
    """(..., d_out) = (act(x w_gate^T) * (x w_up^T)) w_down^T of x (..., d_in)
    with w_gate, w_up (hidden, d_in) and w_down (d_out, hidden), all of one
    type (float32, bfloat16, float16); differentiable with respect to all
    four, once (its gradient has none and says so).  ``activation``: "silu",
    "gelu" (with erf) or "sigmoid".

    Products are summed in float32.  In 16 bits the hidden channels and their
    gradients are held to sixteen bits in float32's range (two bfloat16 pieces),
    so only the outputs are rounded to the type.  A row with an infinite or NaN
    input comes out infinite or NaN, and no other row does."""
    if activation not in _ACTIVATIONS:
        raise ValueError("activation must be 'silu', 'gelu' or 'sigmoid'.")
    if x.ndim < 1 or x.dtype not in _lib.DTYPES:
        raise ValueError("x must be (..., d_in) in float32, bfloat16 or float16.")
    if any(w.dtype != x.dtype for w in (w_gate, w_up, w_down)):
        raise ValueError("x and the weights must have one type.")
    if w_gate.ndim != 2 or w_gate.shape != w_up.shape or w_gate.shape[1] != x.shape[-1]:
        raise ValueError("w_gate and w_up must both have shape (hidden, d_in).")
    if w_down.ndim != 2 or w_down.shape[1] != w_gate.shape[0]:
        raise ValueError("w_down must have shape (d_out, hidden).")
    if min(*w_gate.shape, *w_down.shape) < 1:
        raise ValueError("the block's widths must be at least 1.")
    _lib.check_widths("gsx_ffn_fwd", *w_gate.shape, w_down.shape[0])
    _lib.require_device(x, w_gate, w_up, w_down)
    return _GatedFeedForward.apply(x, w_gate, w_up, w_down, _ACTIVATIONS[activation])


class GatedFeedForward:
    """The block with its weights: ``block(x)`` decodes (..., d_in) rows.

    ``params`` are the leaf tensors ``w_gate``, ``w_up``, ``w_down`` (normal
    with variance 1 / fan-in), as :class:`mlx3d_amd.optim.Adam` takes them."""

    def __init__(self, d_in: int, hidden: int, d_out: int, activation: str = "silu",
                 dtype: torch.dtype = torch.float32, device="cuda", seed: int = 0):
        if min(d_in, hidden, d_out) < 1:
            raise ValueError("the block's widths must be at least 1.")
        if activation not in _ACTIVATIONS:
            raise ValueError("activation must be 'silu', 'gelu' or 'sigmoid'.")
        self.activation = activation
        g = torch.Generator().manual_seed(seed)

        def weight(n_out, n_in):
            w = torch.randn((n_out, n_in), generator=g) / math.sqrt(n_in)
            return w.to(device=device, dtype=dtype).requires_grad_(True)

        self.params = {"w_gate": weight(hidden, d_in), "w_up": weight(hidden, d_in),
                       "w_down": weight(d_out, hidden)}

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        return gated_feed_forward(x, self.params["w_gate"], self.params["w_up"],
                                  self.params["w_down"], self.activation)
