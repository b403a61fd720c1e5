"""Gated feed-forward block, ``(act(x w_gate^T) * (x w_up^T)) w_down^T``, with its gradients (``csrc/kernels/gated.cu``).

Both projections, the activation and the product are one kernel on the tensor cores, the projection back a second one; the
backward pass takes four.  ``float16`` and ``bfloat16``: sums in fp32; ``h``, the result of activation and product, and the
gradients of its two factors are rounded to 16 bits once, as operands of the next product (in ``float16`` what is beyond its
range becomes infinite there).  ``float32``: the products of ``mccl_b200.ops.linear`` (torch's where TF32 is allowed), with one pass
between them; a few tokens without gradients have kernels of their own, in full fp32 whatever is allowed.

What the backward pass needs of the two projections is kept with 16 significant bits (three bytes a number); with
``checkpoint="int8"`` it is kept, and the input too, as 8-bit codes with a scale for each group of 64 (see
``mccl_b200.ops.checkpoint``), and the gradients are those of the kept values (of the input as ``unpack8`` gives it, in its type).  The backward pass is not differentiable itself.
CPU tensors, and calls under a dispatch mode (``make_fx``, flop counters), take the same formulas in torch; a backward pass takes
the form that its forward pass took, and one of the kernels cannot be traced by itself.
"""
from __future__ import annotations

import math
from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F

from ._native import autocast_of, cast, native, without_autocast
from .checkpoint import Packed8, pack8, unpack8

ACTIVATIONS = ("silu", "gelu_tanh")


def gated_feed_forward(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, *,
                       activation: str = "silu", checkpoint: Optional[str] = None) -> torch.Tensor:
    """``x`` [..., width], ``w_gate`` and ``w_up`` [hidden, width], ``w_down`` [width, hidden], all of one type.

    ``activation``: ``"silu"`` or ``"gelu_tanh"``.  ``checkpoint``: ``None`` or ``"int8"``.  Under autocast all four are cast
    to its type first, in every call, as ``torch.nn.functional.linear`` casts them (float64, which the kernels refuse, is not).
    """
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation is one of {ACTIVATIONS}, got {activation!r}")
    if checkpoint not in (None, "int8"):
        raise ValueError(f"checkpoint is None or 'int8', got {checkpoint!r}")
    device = autocast_of(x)
    if device is not None:
        x, w_gate, w_up, w_down = cast(device, x, w_gate, w_up, w_down)
        with torch.autocast(device, enabled=False):
            return _call(x, w_gate, w_up, w_down, activation, checkpoint is not None)
    return _call(x, w_gate, w_up, w_down, activation, checkpoint is not None)


def _call(x, *args):
    y = native()._gated_feed_forward(x, *args) if x.is_cuda else None
    if y is None:
        _check(x, *args[:3])
        *tensors, activation, eight = (x, *args)
        y = _Plain.apply(*tensors, activation, eight and torch.is_grad_enabled() and any(t.requires_grad for t in tensors))
    return y


def _check(x, w_gate, w_up, w_down):
    """Refuses what the kernels refuse, but for types that torch's products take."""
    if any(t.dtype != x.dtype or t.device != x.device for t in (w_gate, w_up, w_down)):
        raise ValueError("gated_feed_forward: tensors differ in type or device")
    if x.dim() < 1 or w_gate.dim() != 2 or w_gate.numel() == 0 or w_up.shape != w_gate.shape or w_down.shape != w_gate.shape[::-1] or x.shape[-1] != w_gate.shape[1]:
        raise ValueError("gated_feed_forward: x [..., width], w_gate and w_up [hidden, width] and w_down [width, hidden] expected, got "
                         + ", ".join(str(tuple(t.shape)) for t in (x, w_gate, w_up, w_down)))


def _act(name, g):
    """The activation and its slope."""
    c = 2 * math.sqrt(2 / math.pi)
    s = torch.sigmoid(g if name == "silu" else c * (g + 0.044715 * g ** 3))
    return g * s, s + g * s * (1 - s) * (1 if name == "silu" else c * (1 + 3 * 0.044715 * g * g))


class _Plain(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, activation, eight):
        g, u = F.linear(x, w_gate), F.linear(x, w_up)
        kept = [pack8(t) for t in (x, g, u)] if eight else [x, g, u]
        ctx.kept_as = [p[2:] for p in kept] if eight else None
        ctx.activation = activation
        ctx.save_for_backward(w_gate, w_up, w_down, *([t for p in kept for t in p[:2]] if eight else kept))
        return F.linear(_act(activation, g)[0] * u, w_down)

    @staticmethod
    @torch.autograd.function.once_differentiable
    @without_autocast
    def backward(ctx, dy):
        w_gate, w_up, w_down, *kept = ctx.saved_tensors
        if ctx.kept_as is not None:
            kept = [unpack8(Packed8(kept[2 * i], kept[2 * i + 1], *ctx.kept_as[i])) for i in range(3)]
        x, g, u = (t.flatten(0, -2) if t.dim() > 1 else t[None] for t in kept)
        rows = dy.reshape(-1, dy.shape[-1])
        a, slope = _act(ctx.activation, g)
        dh = rows @ w_down
        dg, du = dh * u * slope, dh * a
        dx = (dg @ w_gate + du @ w_up).view(dy.shape)
        return dx, dg.t() @ x, du.t() @ x, rows.t() @ (a * u), None, None


class GatedFeedForward(nn.Module):
    """:func:`gated_feed_forward` with its weights, initialised like ``torch.nn.Linear``'s, without biases."""

    def __init__(self, width: int, hidden: int, *, activation: str = "silu", checkpoint: Optional[str] = None, device=None, dtype=None):
        super().__init__()
        if activation not in ACTIVATIONS or checkpoint not in (None, "int8"):
            raise ValueError(f"activation is one of {ACTIVATIONS} and checkpoint None or 'int8'")
        self.activation, self.checkpoint = activation, checkpoint
        like = dict(device=device, dtype=dtype)
        self.w_gate = nn.Parameter(torch.empty(hidden, width, **like))
        self.w_up = nn.Parameter(torch.empty(hidden, width, **like))
        self.w_down = nn.Parameter(torch.empty(width, hidden, **like))
        for w in (self.w_gate, self.w_up, self.w_down):
            nn.init.kaiming_uniform_(w, a=math.sqrt(5))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return gated_feed_forward(x, self.w_gate, self.w_up, self.w_down, activation=self.activation, checkpoint=self.checkpoint)

    def extra_repr(self) -> str:
        hidden, width = self.w_gate.shape
        return f"width={width}, hidden={hidden}, activation={self.activation!r}, checkpoint={self.checkpoint!r}"
