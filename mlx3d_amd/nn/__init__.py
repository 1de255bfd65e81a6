"""Networks over rendered features (hand-written HIP kernels)."""

from .drop import Dropout, dropout  # noqa: F401
from .lookup import Embedding, embedding  # noqa: F401
from .feed_forward import GatedFeedForward, gated_feed_forward  # noqa: F401
from .normalization import LayerNorm, layer_norm  # noqa: F401

__all__ = ["Dropout", "Embedding", "GatedFeedForward", "LayerNorm", "dropout", "embedding",
           "gated_feed_forward", "layer_norm"]
