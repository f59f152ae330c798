"""Optimizers whose step is one launch for many tensors, and the clipping of gradients."""
from .adamw import AdamW
from .clip import clip_grad_norm_

__all__ = ["AdamW", "clip_grad_norm_"]
