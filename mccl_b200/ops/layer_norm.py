"""Layer norm of rows, with the sum with a residual before it, in one pass (``csrc/kernels/norm_forward.cu``, ``norm_backward.cu``).

``y = (s - mean(s)) / sqrt(var(s) + eps) * weight + bias`` along the last dimension, where ``s`` is ``x`` or, with a residual, ``x +
residual`` as the residual's type keeps it; then the sum comes back beside ``y``, and its gradient goes into the one backward pass.  All
in fp32, each result rounded once; float32, float16 and bfloat16.  ``y`` has the type of ``x`` or ``dtype``, so that an fp32
stream can go into 16-bit products without a pass that casts it; autocast changes no types here.

Gradients: of ``x``, the residual (the same numbers, each in its type), the weight and the bias, the last two summed in a fixed order.
The backward pass is not differentiable itself.  CPU tensors, and calls under a dispatch mode (``make_fx``, flop counters), take the
same formulas in torch.
"""
from __future__ import annotations

import math
from typing import Optional

import torch
import torch.nn as nn

from ._native import native

_TYPES = (torch.float32, torch.float16, torch.bfloat16)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *, eps: float = 1e-5,
               residual: Optional[torch.Tensor] = None, dtype: Optional[torch.dtype] = None):
    """``x`` [..., width], ``weight`` and ``bias`` [width] of float32 or of x's type, ``residual`` of x's shape, of float32 or of its type.

    Returns ``y``, or with a residual ``(y, x + residual)``.
    """
    if x.is_cuda:
        out = native()._layer_norm(x, weight, bias, eps, residual, dtype)
        if out is not None:
            return out[0] if residual is None else tuple(out)
    _check(x, weight, bias, eps, residual, dtype)
    return _Plain.apply(x, weight, bias, residual, eps, x.dtype if dtype is None else dtype)


class _Plain(torch.autograd.Function):
    """The formulas in torch."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, eps, dtype):
        s = x if residual is None else (x.float() + residual.float()).to(residual.dtype)
        u = s.float()
        u = u - u.mean(-1, keepdim=True)
        rstd = torch.rsqrt(u.square().mean(-1, keepdim=True) + eps)
        y = u * rstd if weight is None else u * rstd * weight.float()
        ctx.save_for_backward(s, weight, rstd)
        ctx.x_type, ctx.bias_type = x.dtype, None if bias is None else bias.dtype
        ctx.set_materialize_grads(False)
        y = (y if bias is None else y + bias.float()).to(dtype)
        return y if residual is None else (y, s)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, ds=None):
        if dy is None and ds is None:
            return (None,) * 6
        s, weight, rstd = ctx.saved_tensors
        if dy is None:  # the sum's alone: it is x's and the residual's
            none = None if ctx.bias_type is None else torch.zeros(s.shape[-1], dtype=ctx.bias_type, device=s.device)
            return ds.to(ctx.x_type), None if weight is None else torch.zeros_like(weight), none, ds if ctx.needs_input_grad[3] else None, None, None
        u = s.float()
        u = (u - u.mean(-1, keepdim=True)) * rstd
        dy = dy.float()
        g = dy if weight is None else dy * weight.float()
        dx = rstd * (g - g.mean(-1, keepdim=True) - u * (g * u).mean(-1, keepdim=True))
        if ds is not None:
            dx = dx + ds.float()
        rows = tuple(range(dx.dim() - 1))
        total = lambda t, like: (t.sum(rows) if rows else t).to(like)  # noqa: E731
        return (dx.to(ctx.x_type), None if weight is None else total(dy * u, weight.dtype), None if ctx.bias_type is None else total(dy, ctx.bias_type),
                dx.to(s.dtype) if ctx.needs_input_grad[3] else None, None, None)


def _check(x, weight, bias, eps, residual, dtype):
    """Refuses what the kernels refuse."""
    def need(ok, what):
        if not ok:
            raise ValueError(f"layer_norm: {what}")

    need(x.dtype in _TYPES, f"float32, float16 or bfloat16 expected, got {x.dtype}")
    need(x.dim() >= 1 and x.shape[-1] > 0, f"rows of at least one number expected, got {tuple(x.shape)}")
    given = [t for t in (weight, bias) if t is not None]
    need(all(t.shape == x.shape[-1:] and t.is_contiguous() and t.device == x.device and t.dtype in (torch.float32, x.dtype) and t.dtype == given[0].dtype
             for t in given), f"weight and bias are {x.shape[-1]} numbers of float32 or of x's type, on its device, both alike")
    need(residual is None or (residual.shape == x.shape and residual.device == x.device and residual.dtype in (torch.float32, x.dtype)),
         "a residual of x's shape, of float32 or of its type, on its device expected")
    need(dtype is None or dtype in _TYPES, "dtype is float32, float16 or bfloat16")
    need(0 < eps < math.inf, "eps must be positive")


class LayerNorm(nn.LayerNorm):
    """``torch.nn.LayerNorm`` of the last dimension on :func:`layer_norm`."""

    def __init__(self, width: int, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True, device=None, dtype=None):
        super().__init__(width, eps, elementwise_affine, bias, device, dtype)
        if len(self.normalized_shape) != 1:
            raise ValueError(f"LayerNorm is of the last dimension, got {self.normalized_shape}")

    def forward(self, input: torch.Tensor, residual: Optional[torch.Tensor] = None, dtype: Optional[torch.dtype] = None):
        return layer_norm(input, self.weight, self.bias, eps=self.eps, residual=residual, dtype=dtype)
