"""What is measured of the operators inside a decoder block: a gated feed-forward block, the norms and the rotation of
queries and keys, activation checkpoints in 8 bits.

``gated``       ``mccl_b200.ops.gated.gated_feed_forward``: forward alone, or forward and all gradients.
``heads``       ``mccl_b200.ops.heads.norm_rotate`` (separate queries and keys) and ``norm_rotate_packed`` (one projection).
``checkpoint``  ``mccl_b200.ops.checkpoint.pack8`` and ``unpack8``: an activation kept over the forward pass and taken back.

Where ``own`` is false the same formulas run as elementary torch operations in 32 bits, rounded once at the end.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_GROUP = 64         # numbers that share one scale of an 8-bit checkpoint
_TINY = 2.0 ** -100  # a group without a larger number is kept as zeros


def listed():
    return [
        # one token through a block of the width of GPT-2 medium: generation, all latency
        {"name": "gated_token", "kind": "gated", "tokens": 1, "width": 1024, "hidden": 2816, "dtype": "bfloat16",
         "activation": "silu", "grad": False, "checkpoint": False},
        # a short prompt through a block whose hidden width is a multiple of nothing
        {"name": "gated_prompt_odd", "kind": "gated", "tokens": 333, "width": 1000, "hidden": 2731, "dtype": "float16",
         "activation": "gelu_tanh", "grad": False, "checkpoint": False},
        # a training step at the width, sequence and batch of the GPT-2 medium benchmark: 8 sequences of 1024
        {"name": "gated_train", "kind": "gated", "tokens": 8192, "width": 1024, "hidden": 2816, "dtype": "bfloat16",
         "activation": "silu", "grad": True, "checkpoint": False},
        # the same with its activations kept in 8 bits
        {"name": "gated_train_8bit", "kind": "gated", "tokens": 8192, "width": 1024, "hidden": 2816, "dtype": "bfloat16",
         "activation": "silu", "grad": True, "checkpoint": True},
        # a wider block with a larger batch: the largest
        {"name": "gated_train_wide", "kind": "gated", "tokens": 16384, "width": 2048, "hidden": 5632, "dtype": "bfloat16",
         "activation": "gelu_tanh", "grad": True, "checkpoint": False},
        # full precision, the type of the framework's own MLP benchmark, at its batch of 256
        {"name": "gated_train_fp32", "kind": "gated", "tokens": 256, "width": 1024, "hidden": 2816, "dtype": "float32",
         "activation": "silu", "grad": True, "checkpoint": False},
        # one step of generation for 16 sequences with grouped heads
        {"name": "heads_token", "kind": "heads", "batch": 16, "tokens": 1, "heads": 16, "kv_heads": 4, "dim": 64, "rotary": 64,
         "interleaved": False, "packed": True, "dtype": "bfloat16", "grad": False},
        # a training step with the heads of GPT-2 medium: 8 sequences of 1024, 16 heads of 64
        {"name": "heads_train", "kind": "heads", "batch": 8, "tokens": 1024, "heads": 16, "kv_heads": 16, "dim": 64, "rotary": 64,
         "interleaved": False, "packed": True, "dtype": "bfloat16", "grad": True},
        # odd numbers of heads and tokens, a head size with a rotated part, neighbours rotated, separate projections
        {"name": "heads_train_odd", "kind": "heads", "batch": 3, "tokens": 1237, "heads": 6, "kv_heads": 3, "dim": 80, "rotary": 32,
         "interleaved": True, "packed": False, "dtype": "float16", "grad": True},
        # a long document read in at once, grouped heads of 128
        {"name": "heads_long", "kind": "heads", "batch": 1, "tokens": 32768, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128,
         "interleaved": False, "packed": True, "dtype": "bfloat16", "grad": False},
        # a small activation whose last group is ragged
        {"name": "checkpoint_small", "kind": "checkpoint", "rows": 512, "cols": 1000, "dtype": "float32"},
        # the hidden activation of the largest block above
        {"name": "checkpoint_large", "kind": "checkpoint", "rows": 16384, "cols": 5632, "dtype": "bfloat16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["gated", "gated", "heads", "heads", "checkpoint"])
    if kind == "gated":
        dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
        step = rng.choice([1, 8, 64])  # widths that are multiples of nothing, of 16 bytes, of whole tiles
        width = max(step, _log_int(rng, 128, 2048) // step * step)
        hidden = max(step, int(width * rng.uniform(1.5, 4.0)) // step * step)
        grad = rng.random() < 0.6
        tokens = _log_int(rng, 1, 1024 if dtype == "float32" else 8192)
        # (in full precision a code that is rounded the other way shows: the 8-bit form is left to the 16-bit types)
        return {"kind": kind, "tokens": tokens, "width": width, "hidden": hidden, "dtype": dtype,
                "activation": rng.choice(["silu", "gelu_tanh"]), "grad": grad,
                "checkpoint": grad and dtype != "float32" and rng.random() < 0.4}
    if kind == "heads":
        dim = rng.choice([32, 48, 64, 80, 96, 128, 256, 31, 100])
        kv = rng.choice([1, 2, 3, 4, 8])
        tokens = _log_int(rng, 1, 16384)
        return {"kind": kind, "batch": min(rng.choice([1, 2, 3, 8]), max(1, 32768 // tokens)), "tokens": tokens,
                "heads": kv * rng.choice([1, 2, 4]), "kv_heads": kv, "dim": dim,
                "rotary": rng.choice([dim // 2 * 2, dim // 2 * 2, dim // 4 * 2]), "interleaved": rng.random() < 0.4,
                "packed": rng.random() < 0.6, "dtype": rng.choice(["bfloat16", "bfloat16", "float16", "float32"]),
                "grad": rng.random() < 0.6}
    cols = _log_int(rng, 16, 5632)
    return {"kind": kind, "rows": max(1, min(_log_int(rng, 1, 16384), 16384 * 5632 // cols)), "cols": cols,
            "dtype": rng.choice(["bfloat16", "float16", "float32"])}


# ---- inputs --------------------------------------------------------------------------------------
def _device():
    return torch.device("cuda", torch.cuda.current_device())


def _inputs(case, seed):
    """Tensors of one call, on the GPU, from the seed alone."""
    device = _device()
    gen = torch.Generator(device=device)
    gen.manual_seed(int(seed))
    dtype = _DTYPES[case["dtype"]]

    def randn(*shape, std=1.0, to=dtype):
        return (torch.randn(*shape, generator=gen, device=device) * std).to(to)

    kind = case["kind"]
    if kind == "gated":
        m, d, f = case["tokens"], case["width"], case["hidden"]
        # normed activations, weights initialised so that every product keeps their size; gradients of a mean over the tokens
        t = {"x": randn(m, d), "w_gate": randn(f, d, std=d ** -0.5), "w_up": randn(f, d, std=d ** -0.5),
             "w_down": randn(d, f, std=f ** -0.5)}
        if case["grad"]:
            t["dy"] = randn(m, d, std=0.125)
        return t
    if kind == "heads":
        b, n, h, k, d = (case[c] for c in ("batch", "tokens", "heads", "kv_heads", "dim"))
        r = case["rotary"]
        # sequences that begin somewhere in a context of 4096 more tokens
        start = torch.randint(0, 4096, (b, 1), generator=gen, device=device)
        t = {"positions": start + torch.arange(n, device=device)}
        inv = 10000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64, device=device) / r)
        angle = torch.arange(n + 4096, dtype=torch.float64, device=device)[:, None] * inv
        t["table"] = torch.stack((angle.cos(), angle.sin()), 1).float()  # [positions, 2, rotary / 2]
        if case["packed"]:
            t["qkv"] = randn(b, n, (h + 2 * k) * d)
        else:
            t["q"], t["k"] = randn(b, n, h, d), randn(b, n, k, d)
        t["q_weight"] = 1 + randn(d, std=0.2, to=torch.float32)
        t["k_weight"] = 1 + randn(d, std=0.2, to=torch.float32)
        if case["grad"]:
            t["dq"], t["dk"] = randn(b, n, h, d), randn(b, n, k, d)
            if case["packed"]:
                t["dv"] = randn(b, n, k, d)
        return t
    # an activation as it leaves a gated product: heavy tails, a few large channels
    x = torch.randn(case["rows"], case["cols"], generator=gen, device=device)
    x *= torch.randn(case["rows"], case["cols"], generator=gen, device=device)
    x *= torch.exp(torch.randn(case["cols"], generator=gen, device=device))
    return {"x": x.to(dtype)}


def prepare(case, seed):
    t = _inputs(case, seed)
    if case.get("grad"):
        for name in ("x", "w_gate", "w_up", "w_down", "qkv", "q", "k", "q_weight", "k_weight"):
            if name in t:
                t[name].requires_grad_()
    return {"case": case, "t": t}


# ---- one pass ------------------------------------------------------------------------------------
def run(state):
    case, t = state["case"], state["t"]
    kind = case["kind"]
    if own:
        return {"gated": _own_gated, "heads": _own_heads, "checkpoint": _own_checkpoint}[kind](case, t)
    with torch.no_grad():
        return {"gated": _plain_gated, "heads": _plain_heads, "checkpoint": _plain_checkpoint}[kind](case, t)


def _own_gated(case, t):
    from mccl_b200.ops.gated import gated_feed_forward
    args = (t["x"], t["w_gate"], t["w_up"], t["w_down"])
    if not case["grad"]:
        with torch.no_grad():
            return [gated_feed_forward(*args, activation=case["activation"])]
    y = gated_feed_forward(*args, activation=case["activation"], checkpoint="int8" if case["checkpoint"] else None)
    return [y.detach(), *torch.autograd.grad(y, args, t["dy"])]


def _own_heads(case, t):
    from mccl_b200.ops.heads import norm_rotate, norm_rotate_packed
    weights = (t["q_weight"], t["k_weight"])
    if case["packed"]:
        q, k, v = norm_rotate_packed(t["qkv"], *weights, t["table"], t["positions"], heads=case["heads"],
                                     kv_heads=case["kv_heads"], interleaved=case["interleaved"])
        if not case["grad"]:
            return [q, k]
        return [q.detach(), k.detach(), *torch.autograd.grad((q, k, v), (t["qkv"], *weights), (t["dq"], t["dk"], t["dv"]))]
    q, k = norm_rotate(t["q"], t["k"], *weights, t["table"], t["positions"], interleaved=case["interleaved"])
    if not case["grad"]:
        return [q, k]
    return [q.detach(), k.detach(), *torch.autograd.grad((q, k), (t["q"], t["k"], *weights), (t["dq"], t["dk"]))]


def _own_checkpoint(case, t):
    from mccl_b200.ops.checkpoint import pack8, unpack8
    return [unpack8(pack8(t["x"]))]


# ---- the formulas in 32 bits ---------------------------------------------------------------------
def _through_8_bits(x):
    """What comes back of fp32 rows that are kept as codes of 8 bits with a scale for each group."""
    rows, cols = x.shape
    groups = -(-cols // _GROUP)
    v = torch.zeros(rows, groups * _GROUP, device=x.device)
    v[:, :cols] = x
    v = v.view(rows, groups, _GROUP)
    most = v.abs().amax(-1, keepdim=True)
    top = torch.full_like(most, 127.0)
    back = torch.round(v * (top / most)) * (most / top)
    back = torch.where(most < _TINY, torch.zeros_like(back), back)
    back = torch.where(torch.isfinite(most), back, torch.full_like(back, math.nan))
    return back.view(rows, -1)[:, :cols]


def _activation(name, g):
    """The activation and its derivative."""
    if name == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    c = math.sqrt(2 / math.pi)
    th = torch.tanh(c * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1 + th), 0.5 * (1 + th) + 0.5 * g * (1 - th * th) * c * (1 + 3 * 0.044715 * g * g)


def _plain_gated(case, t):
    dtype = t["x"].dtype
    x, wg, wu, wd = (t[k].float() for k in ("x", "w_gate", "w_up", "w_down"))
    g, u = x @ wg.T, x @ wu.T
    y = (_activation(case["activation"], g)[0] * u) @ wd.T
    if not case["grad"]:
        return [y.to(dtype)]
    if case["checkpoint"]:
        x, g, u = _through_8_bits(x), _through_8_bits(g), _through_8_bits(u)
    a, slope = _activation(case["activation"], g)
    dy = t["dy"].float()
    dh = dy @ wd
    dg, du = dh * u * slope, dh * a
    return [r.to(dtype) for r in (y, dg @ wg + du @ wu, dg.T @ x, du.T @ x, dy.T @ (a * u))]


def _pairs(x, rotary, interleaved):
    """The two members of each rotated pair, and what is not rotated."""
    if interleaved:
        return x[..., 0:rotary:2], x[..., 1:rotary:2], x[..., rotary:]
    return x[..., :rotary // 2], x[..., rotary // 2:rotary], x[..., rotary:]


def _join(a, b, rest, interleaved):
    rotated = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((rotated, rest), -1)


def _normed(x, weight, cos, sin, case):
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    a, b, rest = _pairs(x * r * weight, case["rotary"], case["interleaved"])
    return _join(a * cos - b * sin, b * cos + a * sin, rest, case["interleaved"]), r


def _normed_backward(dy, x, r, weight, cos, sin, case):
    a, b, rest = _pairs(dy, case["rotary"], case["interleaved"])
    dn = _join(a * cos + b * sin, b * cos - a * sin, rest, case["interleaved"])
    dx = r * (dn * weight - x * r * r * (dn * weight * x).mean(-1, keepdim=True))
    return dx, (dn * x * r).sum((0, 1, 2))


def _plain_heads(case, t):
    h, k, d = case["heads"], case["kv_heads"], case["dim"]
    if case["packed"]:
        rows = t["qkv"].unflatten(-1, (h + 2 * k, d))
        q, kk = rows[:, :, :h].float(), rows[:, :, h:h + k].float()
        dtype = t["qkv"].dtype
    else:
        q, kk, dtype = t["q"].float(), t["k"].float(), t["q"].dtype
    cs = t["table"][t["positions"]]
    cos, sin = cs[:, :, 0].unsqueeze(2), cs[:, :, 1].unsqueeze(2)
    wq, wk = t["q_weight"], t["k_weight"]
    q1, rq = _normed(q, wq, cos, sin, case)
    k1, rk = _normed(kk, wk, cos, sin, case)
    out = [q1.to(dtype), k1.to(dtype)]
    if not case["grad"]:
        return out
    dq, dwq = _normed_backward(t["dq"].float(), q, rq, wq, cos, sin, case)
    dk, dwk = _normed_backward(t["dk"].float(), kk, rk, wk, cos, sin, case)
    if case["packed"]:
        return out + [torch.cat((dq.to(dtype), dk.to(dtype), t["dv"]), 2).flatten(2), dwq, dwk]
    return out + [dq.to(dtype), dk.to(dtype), dwq, dwk]


def _plain_checkpoint(case, t):
    return [_through_8_bits(t["x"].float()).to(t["x"].dtype)]


# ---- what a pass cannot do without ---------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "gated":
        m, d, f = case["tokens"], case["width"], case["hidden"]
        if not case["grad"]:
            return {"bytes": size * (2 * m * d + 3 * d * f), "flops": 6.0 * m * d * f}
        return {"bytes": size * (4 * m * d + 6 * d * f), "flops": 18.0 * m * d * f}
    if case["kind"] == "heads":
        tokens, d = case["batch"] * case["tokens"], case["dim"]
        rows = tokens * (case["heads"] + case["kv_heads"])
        table = 4 * case["rotary"] * (case["tokens"] + 4096) if tokens > case["tokens"] + 4096 else 4 * case["rotary"] * tokens
        n = 2 * rows * d * size + 8 * tokens + table + 8 * d
        if case["grad"]:
            n += 2 * (rows + (tokens * case["kv_heads"] if case["packed"] else 0)) * d * size + 8 * d
        return {"bytes": n, "flops": rows * d * (24.0 if case["grad"] else 8.0)}
    n = case["rows"] * case["cols"]
    kept = n + 4 * case["rows"] * -(-case["cols"] // _GROUP)
    return {"bytes": 2 * n * size + 2 * kept, "flops": 5.0 * n}


# ---- the definitions in 64 bits ------------------------------------------------------------------
def _kept64(v):
    out = torch.empty_like(v)
    for at in range(0, v.shape[1], _GROUP):
        g = v[:, at:at + _GROUP]
        most = g.abs().max(1, keepdim=True).values
        q = torch.round(g * 127.0 / torch.where(most > 0, most, torch.ones_like(most))) * most / 127.0
        q = torch.where(most < _TINY, torch.zeros_like(q), q)
        out[:, at:at + _GROUP] = torch.where(torch.isfinite(most), q, torch.full_like(q, math.nan))
    return out


def _rotate64(x, angle_cos, angle_sin, rotary, interleaved, back):
    """Rotates by complex multiplication; `back`: the other way."""
    z = torch.complex(*((x[..., 0:rotary:2], x[..., 1:rotary:2]) if interleaved
                        else (x[..., :rotary // 2], x[..., rotary // 2:rotary])))
    w = torch.complex(angle_cos, -angle_sin if back else angle_sin)
    z = z * w
    y = x.clone()
    if interleaved:
        y[..., 0:rotary:2], y[..., 1:rotary:2] = z.real, z.imag
    else:
        y[..., :rotary // 2], y[..., rotary // 2:rotary] = z.real, z.imag
    return y


def exact(case, seed):
    t = {k: v.double() if v.is_floating_point() else v for k, v in _inputs(case, seed).items()}
    if case["kind"] == "checkpoint":
        return [_kept64(t["x"])]
    if case["kind"] == "gated":
        def act(v):
            if case["activation"] == "silu":
                return v * torch.sigmoid(v)
            return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))

        x, wg, wu, wd = t["x"], t["w_gate"], t["w_up"], t["w_down"]
        gate, up = torch.einsum("md,fd->mf", x, wg), torch.einsum("md,fd->mf", x, wu)
        y = torch.einsum("mf,df->md", act(gate) * up, wd)
        if not case["grad"]:
            return [y]
        if case["checkpoint"]:
            x, gate, up = _kept64(x), _kept64(gate), _kept64(up)
        # the derivative from torch's own differentiation of the product, in 64 bits
        with torch.enable_grad():
            gate.requires_grad_(), up.requires_grad_()
            h = act(gate) * up
            d_gate, d_up = torch.autograd.grad(h, (gate, up), torch.einsum("md,df->mf", t["dy"], wd))
        dx = torch.einsum("mf,fd->md", d_gate, wg) + torch.einsum("mf,fd->md", d_up, wu)
        return [y, dx, torch.einsum("mf,md->fd", d_gate, x), torch.einsum("mf,md->fd", d_up, x),
                torch.einsum("md,mf->df", t["dy"], h.detach())]
    h, k, d = case["heads"], case["kv_heads"], case["dim"]
    cs = t["table"][t["positions"]]
    cos, sin = cs[:, :, None, 0], cs[:, :, None, 1]
    if case["packed"]:
        parts = t["qkv"].unflatten(-1, (h + 2 * k, d))
        parts = [parts[:, :, :h], parts[:, :, h:h + k]]
    else:
        parts = [t["q"], t["k"]]
    outs, grads, sums = [], [], []
    for x, w, dy in zip(parts, (t["q_weight"], t["k_weight"]), (t.get("dq"), t.get("dk"))):
        norm = torch.sqrt(x.square().sum(-1, keepdim=True) / d + 1e-6)
        unit = x / norm
        outs.append(_rotate64(unit * w, cos, sin, case["rotary"], case["interleaved"], False))
        if case["grad"]:
            dn = _rotate64(dy, cos, sin, case["rotary"], case["interleaved"], True)
            sums.append((dn * unit).sum((0, 1, 2)))
            dn = dn * w
            grads.append((dn - unit * ((dn * unit).sum(-1, keepdim=True) / d)) / norm)
    if not case["grad"]:
        return outs
    if case["packed"]:
        grads = [torch.cat((*grads, t["dv"]), 2).flatten(2)]
    return [*outs, *grads, *sums]
