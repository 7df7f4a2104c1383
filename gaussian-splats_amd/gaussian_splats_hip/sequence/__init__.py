"""Sequence operators of networks that predict splats from a stream of posed
views, as HIP kernels: the residual norm, a gated linear recurrence and
attention with a sliding window in which the stream's first tokens stay
visible, each for training (forward and backward) and for one token of a
running stream, the attention's cache in the inputs' type or in 4 bits."""

from .attention import (
    WindowCache,
    window_attention,
    window_attention_backward,
    window_attention_forward,
    window_attention_step,
)
from .cache_quant import (
    QuantWindowCache,
    window_attention_step_quant,
    window_cache_fill_quant,
)
from .norm import add_rms_norm, add_rms_norm_backward, add_rms_norm_forward, add_rms_norm_quant
from .scan import gated_scan, gated_scan_backward, gated_scan_forward, gated_scan_step

__all__ = [
    "QuantWindowCache",
    "WindowCache",
    "add_rms_norm",
    "add_rms_norm_backward",
    "add_rms_norm_forward",
    "add_rms_norm_quant",
    "gated_scan",
    "gated_scan_backward",
    "gated_scan_forward",
    "gated_scan_step",
    "window_attention",
    "window_attention_backward",
    "window_attention_forward",
    "window_attention_step",
    "window_attention_step_quant",
    "window_cache_fill_quant",
]
