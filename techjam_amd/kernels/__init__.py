"""HIP kernel entry points (ctypes over the C ABI of ``include/techjam_attn.h``)."""

from .attention import scaled_dot_product_attention, score_guard
from .differential import differential_attention, differential_attention_cached
from .layer_norm import LayerNorm, layer_norm

__all__ = ["LayerNorm", "differential_attention", "differential_attention_cached", "layer_norm",
           "scaled_dot_product_attention", "score_guard"]
