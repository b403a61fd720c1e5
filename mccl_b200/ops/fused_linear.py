"""Linear layer with its bias, an activation and a residual behind the product, ``act(x weight^T + bias) + residual``.

``float16`` and ``bfloat16``, one kernel (and a second one that adds up the parts of tiles whose reduction is shared): the product is on
the tensor cores (``csrc/kernels/gated.cu``, some tens or hundreds of rows ``linear_tiles.cu``), and what follows it is done on its
fp32 sums, rounded once, the activation within 2^-18 of its size, also where the result is ``float32``; a few tokens of which nothing
is kept have a kernel that reads the weights at the rate of memory (``linear_few.cu``).  With a ``float32`` residual, such as the stream
of a model under autocast, the result is ``float32`` too.  ``float32``: the products of ``mccl_b200.ops.linear`` (torch's where it
leaves them to torch or TF32 is allowed), with one pass behind the first and one or two before those of the gradients; small layers
that these would leave to torch's products are whole kernels, in full precision (``linear_small.cu``).

Gradients: of all four.  Behind an activation ``x weight^T + bias`` is kept in the operands' type for the backward pass, which makes
``dz`` of it and of the result's gradient, rounded to that type as an operand of the two products, and the gradient of the bias of
what it was before.  The backward pass is not differentiable itself.  CPU tensors, and calls under a dispatch mode (``make_fx``, flop
counters), take the same formulas in torch.
"""
from __future__ import annotations

import math
from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F

from ._native import autocast_of, cast, native, without_autocast

ACTIVATIONS = (None, "relu", "silu", "gelu", "gelu_tanh")


def fused_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *, activation: Optional[str] = None,
                 residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x`` [..., in], ``weight`` [out, in] and ``bias`` [out] of one type; ``residual`` [..., out] of it or of float32, which the result then is.

    ``activation``: ``None``, ``"relu"``, ``"silu"``, ``"gelu"`` (with the error function) or ``"gelu_tanh"``.  Under autocast the first three
    are cast to its type first, as ``torch.nn.functional.linear`` casts them; the residual stays what it is.
    """
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation is one of {ACTIVATIONS}, got {activation!r}")
    device = autocast_of(x)
    if device is not None:
        x, weight, bias = cast(device, x, weight, bias)
        with torch.autocast(device, enabled=False):
            return _call(x, weight, bias, activation, residual)
    return _call(x, weight, bias, activation, residual)


def _call(x, weight, bias, activation, residual):
    y = native()._fused_linear(x, weight, bias, activation or "none", residual) if x.is_cuda else None
    if y is None:
        _check(x, weight, bias, residual)
        y = _Plain.apply(x, weight, bias, residual, activation)
    return y


def _check(x, weight, bias, residual):
    """Refuses what the kernels refuse, but for types that torch's products take."""
    if any(t is not None and (t.dtype != x.dtype or t.device != x.device) for t in (weight, bias)):
        raise ValueError("fused_linear: tensors differ in type or device")
    if x.dim() < 1 or weight.dim() != 2 or weight.numel() == 0 or x.shape[-1] != weight.shape[1] or (bias is not None and bias.shape != weight.shape[:1]):
        raise ValueError(f"fused_linear: x [..., in], weight [out, in] and bias [out] expected, got {tuple(x.shape)}, {tuple(weight.shape)} and "
                         f"{None if bias is None else tuple(bias.shape)}")
    if residual is not None and (residual.shape != (*x.shape[:-1], weight.shape[0]) or residual.device != x.device
                                 or residual.dtype not in (torch.float32, x.dtype)):
        raise ValueError("fused_linear: a residual of the result's shape, of float32 or of x's type, on its device expected, got "
                         f"{residual.dtype} {tuple(residual.shape)}")


def _act(name, z):
    """The activation and its slope (relu's gradient is no product with one)."""
    if name is None or name == "relu":
        return z if name is None else torch.relu(z), None
    if name == "gelu":
        share = 0.5 * torch.erfc(-z * math.sqrt(0.5))
        return z * share, share + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    c = 2 * math.sqrt(2 / math.pi)
    s = torch.sigmoid(z if name == "silu" else c * (z + 0.044715 * z ** 3))
    return z * s, s + z * s * (1 - s) * (1 if name == "silu" else c * (1 + 3 * 0.044715 * z * z))


def _wide(t):
    return None if t is None else t.float() if t.dtype in (torch.float16, torch.bfloat16) else t


class _Plain(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        z = F.linear(_wide(x), _wide(weight), _wide(bias))
        ctx.activation, ctx.bias = activation, bias is not None
        keep = activation is not None and any(ctx.needs_input_grad[:3])
        kept = z if z.dtype == x.dtype or activation is None else z.clamp(-65504, 65504).to(x.dtype) if x.dtype == torch.float16 else z.to(x.dtype)
        ctx.save_for_backward(x, weight, kept if keep else None)
        ctx.set_materialize_grads(False)
        y = _act(activation, z)[0]
        return y.to(x.dtype) if residual is None else (y + _wide(residual)).to(residual.dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    @without_autocast
    def backward(ctx, dy):
        if dy is None:
            return (None,) * 5
        if not any(ctx.needs_input_grad[:3]):
            return None, None, None, dy, None
        x, weight, z = ctx.saved_tensors
        dz = _wide(dy)
        if z is not None:
            dz = dz.masked_fill(z <= 0, 0) if ctx.activation == "relu" else dz * _act(ctx.activation, _wide(z))[1]
        rows = dz.reshape(-1, dz.shape[-1])
        db = rows.sum(0).to(x.dtype) if ctx.bias else None
        rows = _wide(rows.to(x.dtype))  # an operand of the products
        dx = (rows @ _wide(weight)).to(x.dtype).view(x.shape) if ctx.needs_input_grad[0] else None
        dw = (rows.t() @ _wide(x.reshape(-1, x.shape[-1]))).to(x.dtype) if ctx.needs_input_grad[1] else None
        return dx, dw, db, dy if ctx.needs_input_grad[3] else None, None


class FusedLinear(nn.Linear):
    """``torch.nn.Linear`` on :func:`fused_linear`, with an activation."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, activation: Optional[str] = None, device=None, dtype=None):
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation is one of {ACTIVATIONS}, got {activation!r}")
        super().__init__(in_features, out_features, bias, device, dtype)
        self.activation = activation

    def forward(self, input: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        return fused_linear(input, self.weight, self.bias, activation=self.activation, residual=residual)

    def extra_repr(self) -> str:
        return f"{super().extra_repr()}, activation={self.activation!r}"
