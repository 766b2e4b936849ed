"""Whether a call has to be differentiable."""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

__all__ = ["is_differentiated"]


def is_differentiated(*tensors: torch.Tensor) -> bool:
    """Whether a result computed from ``tensors`` now has to carry a derivative: one of them requires a gradient (and
    gradients are recorded) or is a dual tensor of forward mode. Kernels without a derivative must not take such a call."""
    for t in tensors:
        if t.requires_grad and torch.is_grad_enabled():
            return True
    return forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors)
