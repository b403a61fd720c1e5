"""Decoder of gated feed-forward blocks and normed, rotated heads, on this package's operators.

Per layer: RMS norm, one projection to queries, keys and values, ``ops.heads.norm_rotate_packed``, causal attention with
shared key heads, projection; RMS norm, ``ops.gated``.  ``checkpoint="int8"`` keeps what the gated blocks and the attention's
projections need for their backward pass in 8 bits (``ops.checkpoint``).  Trains like the other models (``wrap_ddp``,
``FusedAdamW``, autocast); :meth:`GatedDecoder.generate` decodes token by token over a cache of keys and values.  In a 16-bit type
(``model.bfloat16()``) a token takes two thirds of what it takes under autocast, which casts the weights in every call.
"""
from __future__ import annotations

import math
from typing import List, Optional, Tuple

import torch
import torch.nn as nn
import torch.nn.functional as F

from ..ops import checkpoint as ckpt
from ..ops.gated import GatedFeedForward
from ..ops.heads import norm_rotate_packed, rotary_table


class _Kept8Linear(nn.Linear):
    """A linear layer that keeps its input in 8 bits."""

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        return ckpt.linear(input, self.weight, self.bias)


class GatedBlock(nn.Module):
    def __init__(self, d: int, heads: int, kv_heads: int, hidden: int, checkpoint: Optional[str]):
        super().__init__()
        if d % heads or heads % kv_heads:
            raise ValueError(f"width {d}, heads {heads} and kv heads {kv_heads} do not divide each other")
        self.heads, self.kv_heads, self.dim, self.checkpoint = heads, kv_heads, d // heads, checkpoint
        linear = _Kept8Linear if checkpoint else nn.Linear
        self.norm1, self.norm2 = nn.RMSNorm(d, eps=1e-6), nn.RMSNorm(d, eps=1e-6)
        self.qkv = linear(d, (heads + 2 * kv_heads) * self.dim, bias=False)
        self.q_norm, self.k_norm = nn.Parameter(torch.ones(self.dim)), nn.Parameter(torch.ones(self.dim))
        self.proj = linear(d, d, bias=False)
        self.ff = GatedFeedForward(d, hidden, checkpoint=checkpoint)

    def forward(self, x, table, positions, cache: Optional[Tuple[torch.Tensor, torch.Tensor]] = None):
        B, T, D = x.shape
        q, k, v = norm_rotate_packed(self.qkv(self.norm1(x)), self.q_norm, self.k_norm, table, positions, heads=self.heads,
                                     kv_heads=self.kv_heads)
        q, k, v = (t.transpose(1, 2) for t in (q, k, v))
        if cache is not None:
            k, v = torch.cat((cache[0], k), 2), torch.cat((cache[1], v), 2)
        # one token sees all of the cache; several at once come with none behind them
        a = F.scaled_dot_product_attention(q, k, v, is_causal=T > 1, enable_gqa=self.heads != self.kv_heads)
        x = x + self.proj(a.transpose(1, 2).reshape(B, T, D))
        return x + self.ff(self.norm2(x)), (k, v)


class GatedDecoder(nn.Module):
    def __init__(self, vocab: int = 50257, d_model: int = 1024, layers: int = 24, heads: int = 16, kv_heads: int = 4, hidden: int = 2816,
                 max_seq: int = 1024, checkpoint: Optional[str] = None):
        super().__init__()
        self.wte = nn.Embedding(vocab, d_model)
        self.blocks = nn.ModuleList(GatedBlock(d_model, heads, kv_heads, hidden, checkpoint) for _ in range(layers))
        self.norm = nn.RMSNorm(d_model, eps=1e-6)
        self.register_buffer("table", rotary_table(max_seq, d_model // heads), persistent=False)
        for name, p in self.named_parameters():
            if p.dim() == 2:  # scaled residual projections, as in GPT-2
                nn.init.normal_(p, std=0.02 / math.sqrt(2 * layers) if name.endswith(("proj.weight", "w_down")) else 0.02)

    def _apply(self, fn, recurse=True):
        table = self.table
        super()._apply(fn, recurse)
        if self.table.dtype != torch.float32:  # cosines of 8 bits are no angles: `to` another type leaves them alone
            self.table = table.to(self.table.device)
        return self

    def _trunk(self, idx, positions, caches: Optional[List] = None):
        x, out = self.wte(idx), []
        for i, b in enumerate(self.blocks):
            x, kv = b(x, self.table, positions, caches[i] if caches else None)
            out.append(kv)
        return self.norm(x), out

    def forward(self, idx, targets=None):
        T = idx.shape[1]
        if T > self.table.shape[0]:
            raise ValueError(f"{T} tokens, and max_seq is {self.table.shape[0]}")
        x, _ = self._trunk(idx, torch.arange(T, device=idx.device))
        logits = F.linear(x, self.wte.weight)  # tied output embedding
        if targets is None:
            return logits
        return F.cross_entropy(logits.view(-1, logits.size(-1)).float(), targets.reshape(-1))

    @torch.no_grad()
    def generate(self, idx, steps: int):
        """``idx`` [batch, tokens] and the ``steps`` most likely next tokens behind it."""
        T = idx.shape[1]
        if T < 1 or T + steps > self.table.shape[0]:
            raise ValueError(f"{T} + {steps} tokens, and max_seq is {self.table.shape[0]}")
        new, caches = idx, None
        for at in range(steps):
            positions = torch.arange(T, device=idx.device) if at == 0 else torch.full((1,), T + at - 1, device=idx.device)
            x, caches = self._trunk(new, positions, caches)
            new = F.linear(x[:, -1:], self.wte.weight).argmax(-1)
            idx = torch.cat((idx, new), 1)
        return idx


def gated_medium(**kw) -> GatedDecoder:
    """GPT-2 medium's width, depth and heads with gated blocks and four key heads."""
    return GatedDecoder(**kw)


def gated_tiny(**kw) -> GatedDecoder:
    """4 layers, d_model 128: the shape used by tests."""
    return GatedDecoder(vocab=kw.pop("vocab", 1024), d_model=128, layers=4, heads=4, kv_heads=2, hidden=352, max_seq=kw.pop("max_seq", 128), **kw)
