"""What the operators with a gradient of their own have in common."""
from __future__ import annotations

from torch.autograd import forward_ad

from ..utils.common import invalidInputError


def refuse_tangents(what: str, *tensors):
    """The kernels have a backward pass only: a tangent of forward-mode differentiation would get lost in silence."""
    if forward_ad._current_level >= 0:
        for t in tensors:
            invalidInputError(t is None or forward_ad.unpack_dual(t).tangent is None,
                              f"{what}: forward-mode gradients are not supported on the GPU")
