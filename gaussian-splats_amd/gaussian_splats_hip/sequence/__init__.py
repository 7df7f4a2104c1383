"""Sequence operators of networks that predict splats from a stream of posed
views, as HIP kernels: the residual norm, a gated linear recurrence and
attention with a sliding window in which the stream's first tokens stay
visible, each for training (forward and backward) and for one token of a
running stream."""

from .norm import add_rms_norm, add_rms_norm_backward, add_rms_norm_forward, add_rms_norm_quant
from .scan import gated_scan, gated_scan_backward, gated_scan_forward, gated_scan_step

__all__ = [
    "add_rms_norm",
    "add_rms_norm_backward",
    "add_rms_norm_forward",
    "add_rms_norm_quant",
    "gated_scan",
    "gated_scan_backward",
    "gated_scan_forward",
    "gated_scan_step",
]
