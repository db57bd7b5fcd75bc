"""Optimizers with native multi-tensor update kernels, and the gradient clipping in front of them."""

from .adamw import AdamW, AdamW8bit
from .clip import clip_grad_norm_, grad_norm

__all__ = ["AdamW", "AdamW8bit", "clip_grad_norm_", "grad_norm"]
