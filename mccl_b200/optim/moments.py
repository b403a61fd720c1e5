"""Moments of an optimizer in 8 bits: floats in units of a power of two that each 256 numbers share (``csrc/kernels/adamw_kinds.cu``).

``exp_avg`` is kept as ``float8_e4m3fn`` and ``exp_avg_sq`` as ``float8_e5m2``, padded to whole groups, with one ``float32`` scale a
group; a value is ``code.float() * scale``.  The largest of a group is at most 1.75 times the format's highest binade.  The optimizer's
step rounds them up or down by chance, so that small changes add up over the steps; :func:`pack_moment`, for a checkpoint's moments, to
nearest.
"""
from __future__ import annotations

import math
from typing import Sequence, Tuple

import torch

GROUP = 256
# digits behind the point, and the exponent of the highest binade used
_FORMS = {torch.float8_e4m3fn: (3, 8), torch.float8_e5m2: (2, 15)}


def padded(numel: int) -> int:
    return -(-numel // GROUP) * GROUP


def pack_moment(x: torch.Tensor, kind: torch.dtype) -> Tuple[torch.Tensor, torch.Tensor]:
    """``x`` in 8 bits: codes of the type ``kind`` and scales.  A group with an infinity or NaN comes back as NaN."""
    digits, top = _FORMS[kind]
    v = torch.zeros(padded(x.numel()), device=x.device)
    v[:x.numel()] = x.detach().reshape(-1)
    v = v.view(-1, GROUP)
    most = v.abs().amax(1, keepdim=True) if v.numel() else v[:, :1]
    power = (((most.view(torch.int32).long() + 0x1FFFFF) >> 23) - 127 - top).clamp(min=-120)
    scale = ((power + 127) << 23).int().view(torch.float32)
    y = v.abs() * ((127 - power) << 23).int().view(torch.float32)
    lowest = 2.0 ** (-6 if digits == 3 else -14)  # below it steps are those of the binade above it
    low = y < lowest
    bits = torch.where(low, y + lowest, y).view(torch.int32).long() + (1 << (22 - digits))
    code = (bits >> (23 - digits)) - (((120 if digits == 3 else 112) + low.long()) << digits)
    if kind is torch.float8_e5m2:  # what divides by its root stays away from zero
        code = torch.where(y > 0, code.clamp(min=1), code)
    else:
        code = code | torch.signbit(v).long() << 7
    finite = torch.isfinite(most)
    code, scale = torch.where(finite, code, 0), torch.where(finite, scale, math.nan)
    return code.to(torch.uint8).view(kind).view(-1), scale.view(-1)


def unpack_moment(codes: torch.Tensor, scale: torch.Tensor, shape: Sequence[int]) -> torch.Tensor:
    """The values as ``float32`` of that shape."""
    return (codes.float().view(-1, GROUP) * scale[:, None]).view(-1)[:math.prod(shape)].view(shape)
