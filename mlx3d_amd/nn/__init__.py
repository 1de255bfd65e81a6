"""Networks over rendered features (hand-written HIP kernels)."""

from .feed_forward import GatedFeedForward, gated_feed_forward  # noqa: F401

__all__ = ["GatedFeedForward", "gated_feed_forward"]
