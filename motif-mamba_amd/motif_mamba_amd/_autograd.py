"""Whether autograd has to see a call. Entry points that go past their autograd function where there is nothing to differentiate
ask here, so that a derivative is either taken or refused, never left out."""
from __future__ import annotations

import torch
from torch.autograd import forward_ad


def differentiated(*tensors):
    """An input requires a gradient, or carries a forward-mode tangent (which needs neither requires_grad nor grad mode; the
    autograd functions refuse it)."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    # Tangents live only within a dual level; without the attribute every tensor is asked.
    if getattr(forward_ad, "_current_level", 0) < 0:
        return False
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)
