"""Activation checkpoints in 8 bits (``csrc/kernels/pack8.cu``).

What a layer keeps from its forward for its backward pass is kept as 8-bit codes, with one fp32 scale for each group of 64
numbers along the last dimension: 1.06 bytes a number.  Of a group, ``scale = max|x| / 127``, ``code = rint(x * (127 /
max|x|))`` and the value that comes back is ``code * scale``: at most half a scale away.  A group that holds an infinity or a
NaN comes back as NaN, so that what went wrong in the forward pass shows in the gradients; a group without a number of 2^-100
comes back as zeros.

:func:`pack8` and :func:`unpack8` are the two halves, for a program's own layers; :func:`linear` is a linear layer whose input
is kept so, and ``mccl_b200.ops.gated`` keeps its activations so on request, written and read inside of its products' kernels.
CPU tensors, and calls under a dispatch mode (``make_fx``, flop counters), take the same formula in torch, bit for bit.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Tuple

import torch
import torch.nn.functional as F

from ._native import autocast_of, cast, native, without_autocast

GROUP = 64
_TINY = 2.0 ** -100
_TYPES = (torch.float32, torch.float16, torch.bfloat16)


class Packed8(NamedTuple):
    """A tensor in 8 bits: ``codes`` (int8, rows padded to 16), ``scales`` (fp32), and the shape and type it had."""
    codes: torch.Tensor
    scales: torch.Tensor
    shape: Tuple[int, ...]
    dtype: torch.dtype


def _check(x: torch.Tensor) -> None:
    if x.dtype not in _TYPES:
        raise TypeError(f"pack8 takes float32, float16 or bfloat16, got {x.dtype}")


def pack8(x: torch.Tensor) -> Packed8:
    """``x`` in 8 bits.  Not differentiable: what is kept is no function of the graph."""
    _check(x)
    if x.is_cuda:
        packed = native()._pack8(x)
        if packed is not None:
            return Packed8(*packed, tuple(x.shape), x.dtype)
    x = x.detach()
    cols = x.shape[-1] if x.dim() else 1
    groups, rows = -(-cols // GROUP), math.prod(x.shape[:-1])
    v = torch.zeros(rows, groups * GROUP, device=x.device)
    v[:, :cols] = x.reshape(rows, cols)
    v = v.view(rows, groups, GROUP)
    most = v.abs().amax(-1, keepdim=True) if v.numel() else v[..., :1]
    top = torch.full_like(most, 127.0)
    keep = (most >= _TINY) & torch.isfinite(most)
    codes = torch.where(keep, torch.round(v * (top / most)), 0.0).view(rows, groups * GROUP)[:, :-(-cols // 16) * 16]
    scales = torch.where(keep, most / top, torch.where(most < _TINY, 0.0, float("nan")))
    return Packed8(codes.to(torch.int8).contiguous(), scales.view(rows, groups), tuple(x.shape), x.dtype)


def unpack8(packed: Packed8) -> torch.Tensor:
    """The values, in the shape and type that they had."""
    if packed.codes.is_cuda:
        x = native()._unpack8(packed.codes, packed.scales, list(packed.shape), packed.dtype)
        if x is not None:
            return x
    cols, rows = packed.shape[-1] if packed.shape else 1, math.prod(packed.shape[:-1])
    if (any(n < 0 for n in packed.shape) or packed.dtype not in _TYPES or packed.codes.dtype != torch.int8 or packed.scales.dtype != torch.float32
            or packed.codes.device != packed.scales.device or packed.codes.shape != (rows, -(-cols // 16) * 16)
            or packed.scales.shape != (rows, -(-cols // GROUP))):
        raise ValueError("unpack8: codes and scales are not those of pack8 for this shape")
    scale = packed.scales.repeat_interleave(GROUP, 1)[:, :cols]
    return (packed.codes[:, :cols].float() * scale).to(packed.dtype).view(packed.shape)


class _Linear8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        kept = pack8(x) if ctx.needs_input_grad[1] else None
        ctx.kept_as = kept and (kept.shape, kept.dtype)
        ctx.save_for_backward(weight, *(kept[:2] if kept else ()))
        return F.linear(x, weight, bias)

    @staticmethod
    @torch.autograd.function.once_differentiable
    @without_autocast
    def backward(ctx, grad):
        weight, *kept = ctx.saved_tensors
        dx = grad.matmul(weight) if ctx.needs_input_grad[0] else None
        rows, dw = grad.reshape(-1, grad.shape[-1]), None
        if ctx.needs_input_grad[1]:
            x = unpack8(Packed8(*kept, *ctx.kept_as))
            dw = rows.t().mm(x.reshape(-1, x.shape[-1]))
        db = rows.sum(0) if ctx.needs_input_grad[2] else None
        return dx, dw, db


def linear(input: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``input @ weight.T + bias``; its input is kept in 8 bits, so the gradient of ``weight`` is that of the kept values.

    Under autocast the three are cast first, as ``torch.nn.functional.linear`` casts them.
    """
    if not torch.is_grad_enabled():  # nothing is kept
        return F.linear(input, weight, bias)
    device = autocast_of(input)
    if device is not None:
        input, weight, bias = cast(device, input, weight, bias)
        with torch.autocast(device, enabled=False):
            return _Linear8.apply(input, weight, bias)
    return _Linear8.apply(input, weight, bias)
