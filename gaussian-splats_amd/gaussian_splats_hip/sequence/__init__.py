"""Sequence operators of networks that predict splats from a stream of posed
views, as HIP kernels: the residual norm, a gated linear recurrence and
attention with a sliding window in which the stream's first tokens stay
visible, each for training (forward and backward) and for one token of a
running stream."""

from .attention import (
    WindowCache,
    window_attention,
    window_attention_backward,
    window_attention_forward,
    window_attention_step,
)
from .norm import add_rms_norm, add_rms_norm_backward, add_rms_norm_forward, add_rms_norm_quant
from .scan import gated_scan, gated_scan_backward, gated_scan_forward, gated_scan_step

__all__ = [
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
]
