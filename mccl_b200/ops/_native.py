"""The native library for operators that torch cannot look into."""
from __future__ import annotations

import functools

import torch

from .. import require_native


def native():
    """The library; refuses under ``torch.jit.trace``, which would record a call's results as constants."""
    if torch._C._get_tracing_state() is not None:
        raise RuntimeError("this operator cannot be traced: it is no operator of torch's")
    return require_native()


def autocast_of(x: torch.Tensor):
    """The device type whose autocast is on for a call on ``x``, or None."""
    device = "cuda" if x.is_cuda else x.device.type
    return device if torch.is_autocast_enabled(device) else None


def cast(device: str, *tensors):
    """The tensors as that autocast casts a product's: float64 stays what it is."""
    to = torch.get_autocast_dtype(device)
    return [t if t is None or t.dtype is torch.float64 else t.to(to) for t in tensors]


def without_autocast(backward):
    """A backward pass whose products are of its tensors' types, also where it is called inside of an autocast region."""
    @functools.wraps(backward)
    def run(ctx, grad):
        device = None if grad is None else autocast_of(grad)
        if device is None:
            return backward(ctx, grad)
        torch.set_autocast_enabled(device, False)
        try:
            return backward(ctx, grad)
        finally:
            torch.set_autocast_enabled(device, True)
    return run
