"""What is measured of the operators of a transformer block's training step: a linear layer with bias, activation and residual in
its product's epilogue, layer norm with the sum before it, and the AdamW step with moments in 8 bits and parameters in 16.

``linear``  ``mccl_b200.ops.fused_linear.fused_linear``: forward alone, or forward and all gradients.
``norm``    ``mccl_b200.ops.layer_norm.layer_norm``: of an activation, or of its sum with a residual, which comes back too.
``adamw``   ``mccl_b200.optim.FusedAdamW`` with ``state_bits=8``, or with 16-bit parameters: one step over a model's tensors.

Where ``own`` is false the same formulas run as elementary torch operations in 32 bits, rounded once at the end.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_GROUP = 256  # moments that share one scale


def listed():
    return [
        # one token through the first layer of a feed-forward block of the width of GPT-2 medium: generation, all latency
        {"name": "linear_token", "kind": "linear", "tokens": 1, "in": 1024, "out": 4096, "dtype": "bfloat16", "activation": "gelu_tanh",
         "residual": "none", "grad": False},
        # a short prompt through a layer whose widths are multiples of nothing
        {"name": "linear_prompt_odd", "kind": "linear", "tokens": 333, "in": 1000, "out": 2731, "dtype": "float16", "activation": "gelu",
         "residual": "same", "grad": False},
        # a training step of GPT-2 medium, 8 sequences of 1024: the first layer of a feed-forward block
        {"name": "linear_train", "kind": "linear", "tokens": 8192, "in": 1024, "out": 4096, "dtype": "bfloat16", "activation": "gelu_tanh",
         "residual": "none", "grad": True},
        # the second one, on a residual stream in fp32, as it is under autocast
        {"name": "linear_train_residual", "kind": "linear", "tokens": 8192, "in": 4096, "out": 1024, "dtype": "bfloat16", "activation": "none",
         "residual": "float32", "grad": True},
        # a wider block with a larger batch: the largest
        {"name": "linear_train_wide", "kind": "linear", "tokens": 16384, "in": 2048, "out": 8192, "dtype": "bfloat16", "activation": "gelu",
         "residual": "none", "grad": True},
        # full precision at the batch of the framework's own MLP benchmark
        {"name": "linear_train_fp32", "kind": "linear", "tokens": 256, "in": 1024, "out": 4096, "dtype": "float32", "activation": "gelu_tanh",
         "residual": "none", "grad": True},
        # one step of generation for 16 sequences
        {"name": "norm_token", "kind": "norm", "rows": 16, "cols": 1024, "dtype": "bfloat16", "residual": "none", "out": "bfloat16", "grad": False},
        # a training step of GPT-2 medium: a projection added to the residual stream, and the norm of the sum
        {"name": "norm_train", "kind": "norm", "rows": 8192, "cols": 1024, "dtype": "bfloat16", "residual": "float32", "out": "bfloat16", "grad": True},
        # odd numbers of rows and columns
        {"name": "norm_train_odd", "kind": "norm", "rows": 4099, "cols": 1723, "dtype": "float16", "residual": "none", "out": "float16", "grad": True},
        # the smallest decoder of the framework: many small tensors
        {"name": "adamw_tiny", "kind": "adamw", "layers": 4, "width": 128, "hidden": 352, "vocab": 1024, "dtype": "float32", "bits": 8},
        # half of the layers of the decoder of GPT-2 medium's width, fp32 parameters
        {"name": "adamw_8bit", "kind": "adamw", "layers": 12, "width": 1024, "hidden": 2816, "vocab": 50257, "dtype": "float32", "bits": 8},
        # the same as a model in bf16
        {"name": "adamw_8bit_bf16", "kind": "adamw", "layers": 12, "width": 1024, "hidden": 2816, "vocab": 50257, "dtype": "bfloat16", "bits": 8},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "norm", "adamw"])
    if kind == "linear":
        dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
        step = rng.choice([1, 8, 64])  # widths that are multiples of nothing, of 16 bytes, of whole tiles
        # (in full precision a sum near zero falls on the other side of relu's corner now and then, and its whole gradient with it)
        activations = ["none", "gelu", "gelu_tanh", "silu"] + (["relu"] if dtype != "float32" else [])
        return {"kind": kind, "tokens": _log_int(rng, 1, 1024 if dtype == "float32" else 8192), "in": max(step, _log_int(rng, 64, 2048) // step * step),
                "out": max(step, _log_int(rng, 64, 4096) // step * step), "dtype": dtype, "activation": rng.choice(activations),
                "residual": rng.choice(["none", "same", "float32"]), "grad": rng.random() < 0.6}
    if kind == "norm":
        cols = _log_int(rng, 16, 8192)
        dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
        residual = rng.choice(["none", "same", "float32"])
        return {"kind": kind, "rows": min(_log_int(rng, 1, 65536), (1 << 24) // cols), "cols": cols, "dtype": dtype, "residual": residual,
                "out": rng.choice([dtype, "bfloat16", "float32"]), "grad": rng.random() < 0.6}
    width = _log_int(rng, 24, 1024)
    dtype = rng.choice(["float32", "bfloat16"])
    return {"kind": kind, "layers": rng.randint(1, 8), "width": width, "hidden": int(width * rng.uniform(1.5, 4.0)), "vocab": _log_int(rng, 100, 50257),
            "dtype": dtype, "bits": 8 if dtype == "float32" else rng.choice([8, 8, 32])}


# ---- inputs --------------------------------------------------------------------------------------
def _device():
    return torch.device("cuda", torch.cuda.current_device())


def _type_of(case, what):
    """The type of the residual, and of what is added to it: None without one."""
    return None if case[what] == "none" else _DTYPES[case["dtype"] if case[what] == "same" else case[what]]


def _sizes(case):
    """The tensors of a decoder: embedding, and of each layer projections, gated block, norms."""
    d, f = case["width"], case["hidden"]
    return [case["vocab"] * d] + [3 * d // 2 * d, d * d, f * d, f * d, d * f, d, d, 64, 64] * case["layers"] + [d]


def _power(most, top):
    """The power of two that takes the largest of a group to at most 1.75 * 2^top."""
    most = torch.clamp(most, 1e-30, 1e30)
    return torch.exp2(torch.ceil(torch.log2(most / 1.75)) - top)


def _inputs(case, seed):
    """Tensors of one call, on the GPU, from the seed alone."""
    device = _device()
    gen = torch.Generator(device=device)
    gen.manual_seed(int(seed))
    dtype = _DTYPES[case["dtype"]]

    def randn(*shape, std=1.0, to=dtype):
        return (torch.randn(*shape, generator=gen, device=device) * std).to(to)

    if case["kind"] == "linear":
        m, k, n = case["tokens"], case["in"], case["out"]
        stream = _type_of(case, "residual")
        # normed activations, weights that keep their size; gradients of a mean over the tokens
        t = {"x": randn(m, k), "weight": randn(n, k, std=k ** -0.5), "bias": randn(n, std=0.1)}
        if stream is not None:
            t["residual"] = randn(m, n, std=2.0, to=stream)
        if case["grad"]:
            t["dy"] = randn(m, n, std=0.125, to=stream or dtype)
        return t
    if case["kind"] == "norm":
        rows, cols = case["rows"], case["cols"]
        stream = _type_of(case, "residual")
        # a residual stream has a mean, and a few channels much larger than the others
        channel = torch.exp(torch.randn(cols, generator=gen, device=device)) + 0.25
        t = {"x": ((torch.randn(rows, cols, generator=gen, device=device) + 0.3) * channel).to(dtype)}
        if stream is not None:
            t["residual"] = ((torch.randn(rows, cols, generator=gen, device=device) + 0.3) * channel).to(stream)
        t["weight"] = 1 + randn(cols, std=0.2, to=torch.float32)
        t["bias"] = randn(cols, std=0.1, to=torch.float32)
        if case["grad"]:
            t["dy"] = randn(rows, cols, to=_DTYPES[case["out"]])
            if stream is not None:
                t["ds"] = randn(rows, cols, to=stream)
        return t
    # every tensor begins a new group in buffers that hold all of them, and what is between them stays zero
    sizes = _sizes(case)
    starts, n = [], 0
    for size in sizes:
        starts.append(n)
        n += -(-size // _GROUP) * _GROUP
    used = torch.zeros(n, dtype=torch.bool, device=device)
    for at, size in zip(starts, sizes):
        used[at:at + size] = True
    spread = torch.exp(torch.randn(n, generator=gen, device=device)) * 1e-3
    noise = torch.randn(n, generator=gen, device=device)
    grad = spread * torch.randn(n, generator=gen, device=device) * used
    # moments of some thousand steps: a mean of gradients a third of their size, a mean of their squares
    first = (spread * noise * 0.3 * used).view(-1, _GROUP)
    second = (spread * spread * (1 + 0.2 * noise.abs()) * used).view(-1, _GROUP)
    t = {"grad": grad.to(dtype), "param": randn(n, std=0.02) * used}
    if case["bits"] == 8:
        for name, moment, top, kind in (("exp_avg", first, 8, torch.float8_e4m3fn), ("exp_avg_sq", second, 15, torch.float8_e5m2)):
            scale = _power(moment.abs().amax(1, keepdim=True), top)
            t[name] = (moment / scale).to(kind).view(-1)
            t[name + "_scale"] = scale.view(-1)
    else:
        t["exp_avg"], t["exp_avg_sq"] = first.reshape(-1).contiguous(), second.reshape(-1).contiguous()
    if dtype is torch.bfloat16:
        t["low"] = torch.randint(-32768, 32768, (n,), generator=gen, device=device, dtype=torch.int16) * used
    # which number of its own tensor each is
    t["index"] = torch.arange(n, dtype=torch.int32, device=device)
    for at, size in zip(starts, sizes):
        t["index"][at:at + size] -= at
    return {**t, "starts": starts, "sizes": sizes, "step": 1000}


def prepare(case, seed):
    t = _inputs(case, seed)
    if case["kind"] != "adamw":
        if case["grad"]:
            for name in ("x", "weight", "bias", "residual"):
                if name in t:
                    t[name].requires_grad_()
        return {"case": case, "t": t}
    params, states = [], []
    for at, size in zip(t["starts"], t["sizes"]):
        p = torch.nn.Parameter(t["param"][at:at + size])
        p.grad = t["grad"][at:at + size]
        whole, groups = slice(at, at + -(-size // _GROUP) * _GROUP), slice(at // _GROUP, at // _GROUP + -(-size // _GROUP))
        state = {"step": torch.tensor(float(t["step"]))}
        for name in ("exp_avg", "exp_avg_sq"):
            if case["bits"] == 8:
                state[name], state[name + "_scale"] = t[name][whole], t[name + "_scale"][groups]
            else:
                state[name] = t[name][at:at + size]
        if "low" in t:
            state["low"] = t["low"][at:at + size]
        params.append(p)
        states.append(state)
    state = {"case": case, "t": t}
    if own:  # the optimizer that a program keeps, as it is after loading a checkpoint
        from mccl_b200.optim import FusedAdamW
        state["optimizer"] = FusedAdamW(params, lr=1e-3, state_bits=case["bits"])
        for p, s in zip(params, states):
            state["optimizer"].state[p] = s
    return state


# ---- one pass ------------------------------------------------------------------------------------
def run(state):
    case, t = state["case"], state["t"]
    kind = case["kind"]
    if own:
        return {"linear": _own_linear, "norm": _own_norm, "adamw": _own_adamw}[kind](case, t, state)
    with torch.no_grad():
        return {"linear": _plain_linear, "norm": _plain_norm, "adamw": _plain_adamw}[kind](case, t)


def _own_linear(case, t, _):
    from mccl_b200.ops.fused_linear import fused_linear
    leaves = [t[name] for name in ("x", "weight", "bias", "residual") if name in t]
    call = dict(activation=None if case["activation"] == "none" else case["activation"], residual=t.get("residual"))
    if not case["grad"]:
        with torch.no_grad():
            return [fused_linear(*leaves[:3], **call)]
    y = fused_linear(*leaves[:3], **call)
    return [y.detach(), *torch.autograd.grad(y, leaves, t["dy"])]


def _own_norm(case, t, _):
    from mccl_b200.ops.layer_norm import layer_norm
    leaves = [t[name] for name in ("x", "weight", "bias", "residual") if name in t]
    if not case["grad"]:
        with torch.no_grad():
            out = layer_norm(*leaves[:3], residual=t.get("residual"), dtype=_DTYPES[case["out"]])
        return list(out) if "residual" in t else [out]
    out = layer_norm(*leaves[:3], residual=t.get("residual"), dtype=_DTYPES[case["out"]])
    if "residual" in t:
        return [*(o.detach() for o in out), *torch.autograd.grad(out, leaves, (t["dy"], t["ds"]))]
    return [out.detach(), *torch.autograd.grad(out, leaves, t["dy"])]


def _moments_of(case, t):
    # (moments in 8 bits as 8-bit floats, which are the values in units of their group's scale)
    names = ["exp_avg", "exp_avg_sq"] + (["exp_avg_scale", "exp_avg_sq_scale"] if case["bits"] == 8 else [])
    return [t["param"], *(t[name] for name in names), *([t["low"]] if "low" in t else [])]


def _own_adamw(case, t, state):
    state["optimizer"].step()
    return _moments_of(case, t)


# ---- the formulas in 32 bits ---------------------------------------------------------------------
def _activation(name, z):
    """The activation and its derivative."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z)), (z > 0).float()
    if name == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    if name == "gelu":
        share = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * share, share + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    c = math.sqrt(2 / math.pi)
    th = torch.tanh(c * (z + 0.044715 * z * z * z))
    return 0.5 * z * (1 + th), 0.5 * (1 + th) + 0.5 * z * (1 - th * th) * c * (1 + 3 * 0.044715 * z * z)


def _plain_linear(case, t):
    dtype = t["x"].dtype
    x, w, bias = (t[k].float() for k in ("x", "weight", "bias"))
    a, slope = _activation(case["activation"], x @ w.T + bias)
    y = (a + t["residual"].float()).to(t["residual"].dtype) if "residual" in t else a.to(dtype)
    if not case["grad"]:
        return [y]
    dz = t["dy"].float() * slope
    return [y, (dz @ w).to(dtype), (dz.T @ x).to(dtype), dz.sum(0).to(dtype), *([t["dy"]] if "residual" in t else [])]


def _plain_norm(case, t):
    s, out = t["x"].float(), _DTYPES[case["out"]]
    if "residual" in t:
        kept = (s + t["residual"].float()).to(t["residual"].dtype)
        s = kept.float()
    s = s - s.mean(-1, keepdim=True)
    r = 1 / torch.sqrt((s * s).mean(-1, keepdim=True) + 1e-5)
    unit = s * r
    y = (unit * t["weight"] + t["bias"]).to(out)
    result = [y, kept] if "residual" in t else [y]
    if not case["grad"]:
        return result
    dy = t["dy"].float()
    g = dy * t["weight"]
    dx = r * (g - g.mean(-1, keepdim=True) - unit * (g * unit).mean(-1, keepdim=True))
    sums = [(dy * unit).sum(0), dy.sum(0)]
    if "residual" in t:
        dx = dx + t["ds"].float()
        return [*result, dx.to(t["x"].dtype), *sums, dx.to(t["residual"].dtype)]
    return [*result, dx.to(t["x"].dtype), *sums]


def _dither(index, step):
    """Two whole numbers of 16 bits for each number of a tensor and each step."""
    word = 0xFFFFFFFF
    h = ((index.long() ^ (step * 0x9E3779B9 & word)) * 0x6A09E667) & word
    h ^= h >> 15
    h = (h * 0xBB67AE85) & word
    h ^= h >> 16
    return h & 0xFFFF, h >> 16


def _bits(x):
    return x.view(torch.int32).long()


def _to_codes(x, dither, top, digits, positive):
    """Groups of fp32 numbers as 8-bit floats of so many digits behind the point, rounded up as often as the dither says, and scales."""
    small, bias = (2.0 ** -6, 120) if digits == 3 else (2.0 ** -14, 112)
    most = x.abs().amax(1, keepdim=True)
    power = torch.clamp(((_bits(most) + 0x1FFFFF) >> 23) - 127 - top, min=-120)
    scale = ((power + 127) << 23).int().view(torch.float32)
    y = x.abs() * ((127 - power) << 23).int().view(torch.float32)
    low = y < small
    z = torch.where(low, y + torch.full_like(y, small), y)
    code = ((_bits(z) + (dither << (7 - digits))) >> (23 - digits)) - ((bias + low.long()) << digits)
    if positive:
        code = torch.where(y > 0, torch.clamp(code, min=1), code)
    else:
        code = code | (torch.signbit(x).long() << 7)
    finite = torch.isfinite(most)
    code = torch.where(finite, code, torch.zeros_like(code))
    return code.to(torch.uint8), torch.where(finite, scale, torch.full_like(scale, math.nan))


def _plain_adamw(case, t):
    lr, b1, b2, eps, decay = 1e-3, 0.9, 0.999, 1e-8, 1e-2
    t["step"] += 1
    step, eight, half = t["step"], case["bits"] == 8, "low" in t
    g = t["grad"].float()
    m, v = t["exp_avg"].float(), t["exp_avg_sq"].float()
    if eight:
        m = (m.view(-1, _GROUP) * t["exp_avg_scale"][:, None]).view(-1)
        v = (v.view(-1, _GROUP) * t["exp_avg_sq_scale"][:, None]).view(-1)
    p = t["param"]
    if half:  # the upper 16 bits of a float, and what they leave
        low = torch.where((p == 0) & (t["low"] < 0), torch.zeros_like(t["low"]), t["low"])
        p = ((p.view(torch.int16).int() << 16) + low.int()).view(torch.float32)
    p = p * (1 - lr * decay)
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * (1 - b2) * g
    p = p - m / (torch.sqrt(v) * (1 / math.sqrt(1 - b2 ** step)) + eps) * (lr / (1 - b1 ** step))
    if half:
        bits = _bits(p)
        upper = torch.where(torch.isnan(p), torch.full_like(bits, 0x7FC0), (bits + 0x8000) >> 16)
        t["low"].copy_(torch.where(torch.isnan(p), torch.zeros_like(bits), bits - (upper << 16)))
        t["param"].copy_(upper.to(torch.int16).view(torch.bfloat16))
    else:
        t["param"].copy_(p)
    if eight:
        dither = _dither(t["index"], step)
        for name, moment, rest in (("exp_avg", m, (8, 3, False)), ("exp_avg_sq", v, (15, 2, True))):
            code, scale = _to_codes(moment.view(-1, _GROUP), dither[rest[2]].view(-1, _GROUP), *rest)
            t[name].view(torch.uint8).copy_(code.view(-1))
            t[name + "_scale"].copy_(scale.view(-1))
    else:
        t["exp_avg"].copy_(m)
        t["exp_avg_sq"].copy_(v)
    return _moments_of(case, t)


# ---- what a pass cannot do without ---------------------------------------------------------------
def work(case):
    size = {"float32": 4, "bfloat16": 2, "float16": 2}
    own_size = size[case["dtype"]]
    if case["kind"] == "adamw":
        n = float(sum(_sizes(case)))
        moments = 4 * (1 + 4 / _GROUP) if case["bits"] == 8 else 16
        return {"bytes": n * (moments + 3 * own_size + (4 if case["dtype"] == "bfloat16" else 0)), "flops": 15 * n}
    stream = 0 if case["residual"] == "none" else own_size if case["residual"] == "same" else size[case["residual"]]
    if case["kind"] == "linear":
        m, k, n = case["tokens"], case["in"], case["out"]
        out = stream or own_size
        if not case["grad"]:
            return {"bytes": own_size * (m * k + n * k + n) + m * n * (out + stream), "flops": 2.0 * m * k * n}
        return {"bytes": own_size * 2 * (m * k + n * k + n) + m * n * (2 * out + stream), "flops": 6.0 * m * k * n}
    rows, cols, out = case["rows"], case["cols"], size[case["out"]]
    n = rows * cols * (own_size + 2 * stream + out) + 8 * cols
    if case["grad"]:
        n += rows * cols * (own_size + (2 if case["residual"] == "float32" else 1) * stream + out) + 8 * cols
    return {"bytes": float(n), "flops": rows * cols * (24.0 if case["grad"] else 8.0)}


# ---- the definitions in 64 bits ------------------------------------------------------------------
def exact(case, seed):
    t = _inputs(case, seed)
    if case["kind"] == "adamw":
        m, v = t["exp_avg"].double(), t["exp_avg_sq"].double()
        if case["bits"] == 8:
            m *= t["exp_avg_scale"].double().repeat_interleave(_GROUP)
            v *= t["exp_avg_sq_scale"].double().repeat_interleave(_GROUP)
        p, g, step = t["param"].double(), t["grad"].double(), t["step"] + 1
        if "low" in t:  # a float's upper bits and what they leave of it, as one whole number
            p = (t["param"].view(torch.int16).to(torch.int32) * 65536 + t["low"]).view(torch.float32).double()
        m.lerp_(g, 0.1)
        v.lerp_(g.square_(), 0.001)
        p = p * (1 - 1e-5) - 1e-3 * (m / (1 - 0.9 ** step)) / ((v / (1 - 0.999 ** step)).sqrt_() + 1e-8)
        # how the moments are rounded, and what a 16-bit parameter leaves of itself, has no value apart from the fp32 formula
        moments = [None] * 4 if case["bits"] == 8 else [m, v]
        return [p, *moments] + ([None] if "low" in t else [])
    if case["kind"] == "linear":
        x, w, bias = (t[k].double() for k in ("x", "weight", "bias"))
        with torch.enable_grad():  # the derivative from torch's own differentiation, in 64 bits
            z = torch.einsum("mk,nk->mn", x, w).add_(bias).requires_grad_()
            a = {"none": lambda z: z * 1.0, "relu": torch.relu, "silu": lambda z: z * torch.sigmoid(z),
                 "gelu": lambda z: z * torch.special.ndtr(z),
                 "gelu_tanh": lambda z: 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))}[case["activation"]](z)
            if case["grad"]:
                (dz,) = torch.autograd.grad(a, z, t["dy"].double())
        y = a.detach()
        if "residual" in t:
            y = y + t["residual"].double()
        if not case["grad"]:
            return [y]
        return [y, torch.einsum("mn,nk->mk", dz, w), torch.einsum("mn,mk->nk", dz, x), torch.einsum("mn->n", dz),
                *([t["dy"].double()] if "residual" in t else [])]
    s = t["x"].double()
    if "residual" in t:  # the sum is kept in the stream's type, and what is normed is what is kept
        s = (s + t["residual"].double()).to(t["residual"].dtype).double()
    with torch.enable_grad():
        leaf, weight, bias = s.clone().requires_grad_(), t["weight"].double().requires_grad_(), t["bias"].double().requires_grad_()
        deviation, mean = torch.var_mean(leaf, -1, correction=0, keepdim=True)
        y = torch.addcmul(bias, (leaf - mean) * (deviation + 1e-5).rsqrt(), weight)
        result = [y.detach(), s] if "residual" in t else [y.detach()]
        if not case["grad"]:
            return result
        dx, dw, db = torch.autograd.grad(y, (leaf, weight, bias), t["dy"].double())
    if "residual" in t:
        dx = dx + t["ds"].double()
        return [*result, dx, dw, db, dx]
    return [*result, dx, dw, db]
