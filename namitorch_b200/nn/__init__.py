"""``namitorch_b200.nn.functional`` holds the fused cross-entropy of the hot path,
sliding-window attention and counter-based dropout."""
from . import functional

__all__ = ["functional"]
