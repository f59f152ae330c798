"""Optimizers whose step is one launch for many tensors."""
from .adamw import AdamW

__all__ = ["AdamW"]
