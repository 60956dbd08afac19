"""What the operators with a gradient of their own have in common."""
from __future__ import annotations

import contextlib

import torch
from torch.autograd import forward_ad

from ..utils.common import invalidInputError


_HERE = contextlib.nullcontext()


def on(dev: torch.device):
    """A guard for launches on another device than the current one."""
    return _HERE if torch._C._cuda_getDevice() == dev.index else torch.cuda.device(dev)


def refuse_tangents(what: str, *tensors):
    """The kernels have a backward pass only: a tangent of forward-mode differentiation would get lost in silence."""
    if forward_ad._current_level >= 0:
        for t in tensors:
            invalidInputError(t is None or forward_ad.unpack_dual(t).tangent is None,
                              f"{what}: forward-mode gradients are not supported on the GPU")
