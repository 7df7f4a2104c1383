"""Training-step pieces that consume the rendered image: the loss terms of
the reference's training step, its optimiser and the clipping of its gradients'
norm, as HIP kernels."""

from .clip import clip_grad_norm, grad_norm
from .losses import (
    l1_loss,
    l1_loss_backward,
    l1_loss_forward,
    splat_regularizers,
    ssim,
    ssim_backward,
    ssim_forward,
)
from .optim import FusedAdam

__all__ = [
    "FusedAdam",
    "clip_grad_norm",
    "grad_norm",
    "l1_loss",
    "l1_loss_backward",
    "l1_loss_forward",
    "splat_regularizers",
    "ssim",
    "ssim_backward",
    "ssim_forward",
]
