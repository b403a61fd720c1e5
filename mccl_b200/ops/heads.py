"""Norms of queries and keys for each head, and the rotation by position, in one pass (``csrc/kernels/heads.cu``).

Of each row ``x`` of one head of one token: ``n = x / sqrt(mean(x^2) + eps) * weight``; the first ``rotary`` numbers of ``n``
are pairs, ``(i, i + rotary / 2)`` or, ``interleaved``, ``(2 i, 2 i + 1)``, each rotated by its angle of the token's position:
``a' = a cos - b sin``, ``b' = b cos + a sin``.  All in fp32, rounded once; float32, float16 and bfloat16, head sizes up to 512.

The angles come from a table, :func:`rotary_table` or a program's own (scaled or interpolated ones), float32 ``[positions, 2,
rotary / 2]``, cosines and then sines.  A token whose position is outside of the table gets NaN in its rotated part.

Gradients: of queries and keys (of the packed form one gradient of the projection, values included) and of the two weights,
summed in a fixed order.  The backward pass is not differentiable itself.  CPU tensors, and calls under a dispatch mode
(``make_fx``, flop counters), take the same formulas in torch.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from ._native import native

_TYPES = (torch.float32, torch.float16, torch.bfloat16)


def rotary_table(positions: int, rotary: int, *, theta: float = 10000.0, device=None) -> torch.Tensor:
    """Cosines and sines of ``position * theta^(-2 i / rotary)``, computed in 64 bits: ``[positions, 2, rotary / 2]``."""
    if rotary < 0 or rotary % 2 or positions < 0:
        raise ValueError(f"rotary_table needs an even rotary size and a number of positions, got {rotary} and {positions}")
    turn = theta ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=device) / max(rotary, 1))
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * turn
    return torch.stack((angle.cos(), angle.sin()), 1).float()


def norm_rotate(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, table: torch.Tensor,
                positions: Optional[torch.Tensor] = None, *, eps: float = 1e-6,
                interleaved: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """``q`` [batch, tokens, heads, dim] and ``k`` [batch, tokens, kv heads, dim], normed and rotated, contiguous.

    ``positions``: int64 or int32, [tokens] or [batch, tokens]; 0, 1, ... in each batch without it.
    """
    if q.is_cuda:
        out = native()._norm_rotate(q, k, q_weight, k_weight, table, positions, eps, interleaved)
        if out is not None:
            return out
    _check(q, k, q_weight, k_weight, table, positions, eps)
    return (_plain(q, q_weight, table, positions, eps, interleaved), _plain(k, k_weight, table, positions, eps, interleaved))


def norm_rotate_packed(qkv: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, table: torch.Tensor,
                       positions: Optional[torch.Tensor] = None, *, heads: int, kv_heads: Optional[int] = None,
                       eps: float = 1e-6, interleaved: bool = False) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """:func:`norm_rotate` of one projection [batch, tokens, (heads + 2 kv_heads) * dim]; also the view of its values."""
    kv_heads = heads if kv_heads is None else kv_heads
    if qkv.is_cuda:
        out = native()._norm_rotate_packed(qkv, q_weight, k_weight, table, positions, heads, kv_heads, eps, interleaved)
        if out is not None:
            return out
    if qkv.dim() != 3 or heads < 1 or kv_heads < 1 or qkv.shape[-1] % (heads + 2 * kv_heads):
        raise ValueError(f"norm_rotate_packed: [batch, tokens, (heads + 2 kv_heads) dim] expected, got {tuple(qkv.shape)}")
    q, k, v = qkv.unflatten(-1, (heads + 2 * kv_heads, -1)).split((heads, kv_heads, kv_heads), 2)
    q, k = norm_rotate(q, k, q_weight, k_weight, table, positions, eps=eps, interleaved=interleaved)
    return q, k, v


def _check(q, k, q_weight, k_weight, table, positions, eps):
    """Refuses what the kernels refuse."""
    def need(ok, what):
        if not ok:
            raise ValueError(f"norm_rotate: {what}")

    need(q.dim() == 4 and k.dim() == 4 and q.shape[:2] == k.shape[:2] and q.shape[3] == k.shape[3] and q.shape[2] > 0 and k.shape[2] > 0,
         f"queries [batch, tokens, heads, dim] and keys [batch, tokens, kv heads, dim] expected, got {tuple(q.shape)} and {tuple(k.shape)}")
    dim, alike = q.shape[3], lambda t: t.device == q.device
    need(q.dtype in _TYPES and k.dtype == q.dtype and alike(k), "queries and keys of one of float32, float16 and bfloat16 on one device expected")
    need(0 < dim <= 512, f"head sizes up to 512, got {dim}")
    need(all(w.shape == (dim,) and w.is_contiguous() and alike(w) and w.dtype == q_weight.dtype for w in (q_weight, k_weight))
         and q_weight.dtype in (torch.float32, q.dtype), f"weights are {dim} numbers of float32 or of the queries' type, on their device, both alike")
    need(table.dim() == 3 and table.shape[1] == 2 and table.dtype == torch.float32 and table.is_contiguous() and alike(table)
         and not table.requires_grad and 2 * table.shape[2] <= dim,
         f"a contiguous float32 table [positions, 2, rotary / 2] without gradient expected, rotary at most {dim}")
    need(0 < eps < math.inf, "eps must be positive")
    need(positions is None or (positions.dtype in (torch.int64, torch.int32) and alike(positions) and positions.dim() in (1, 2)
                               and positions.shape[-1] == q.shape[1] and (positions.dim() == 1 or positions.shape[0] in (1, q.shape[0]))),
         "positions are int64 or int32, [tokens] or [batch, tokens]")


def _plain(x, weight, table, positions, eps, interleaved):
    if positions is None:
        positions = torch.arange(x.shape[1], device=x.device)
    inside = (positions >= 0) & (positions < table.shape[0])
    if table.shape[0] == 0:  # all are outside; a row to look them up in
        table = table.new_zeros((1, *table.shape[1:]))
    cs = table[positions.clamp(0, table.shape[0] - 1).long()].masked_fill(~inside[..., None, None], float("nan"))
    cos, sin = cs[..., None, 0, :], cs[..., None, 1, :]   # one head for all
    half = table.shape[-1]
    n = x.float()
    n = n * torch.rsqrt(n.square().mean(-1, keepdim=True) + eps) * weight.float()
    a, b = (n[..., 0:2 * half:2], n[..., 1:2 * half:2]) if interleaved else (n[..., :half], n[..., half:2 * half])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((turned, n[..., 2 * half:]), -1).to(x.dtype)
