"""The linear layer with bias, activation and residual against its formulas in 64 bits."""
import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils.flop_counter import FlopCounterMode

from mccl_b200.ops.fused_linear import FusedLinear, fused_linear

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
ROUNDOFF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
U = 2.0 ** -24
ACTIVATIONS = [None, "relu", "silu", "gelu", "gelu_tanh"]


def _act(name, z):
    if name is None:
        return z, torch.ones_like(z)
    if name == "relu":
        return torch.relu(z), (z > 0).to(z.dtype)
    if name == "gelu":
        return z * torch.special.ndtr(z), torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    c = 2 * math.sqrt(2 / math.pi)
    s = torch.sigmoid(z if name == "silu" else c * (z + 0.044715 * z ** 3))
    return z * s, s + z * s * (1 - s) * (1 if name == "silu" else c * (1 + 3 * 0.044715 * z * z))


def _sum(dtype, depth):
    """Products of 16-bit numbers are exact in fp32; the tensor cores cut each sum of (at least) 8 of them off at 2^-23 of what it adds
    up.  fp32 products are six bf16 products (2^-20) or sums of a library kernel (2^-24 a term)."""
    return (depth / 8 + 4) * 2.0 ** -23 if dtype != torch.float32 else 2.0 ** -20 + (depth + 2) * U


def _inputs(tokens, width, out, dtype, residual, bias, device, seed=0, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    t = {"x": (randn(tokens, width) * scale).to(dtype), "weight": (randn(out, width) * width ** -0.5).to(dtype)}
    if bias:
        t["bias"] = (randn(out) * 0.5).to(dtype)
    if residual is not None:
        t["residual"] = (2 * randn(tokens, out)).to(residual)
    t["dy"] = randn(tokens, out).to(residual or dtype)
    return {k: v.to(device) for k, v in t.items()}


def _leaves(t):
    return [t[k] for k in ("x", "weight", "bias", "residual") if k in t]


def _call(t, activation, grad=True):
    if not grad:
        return [fused_linear(t["x"].detach(), t["weight"].detach(), None if "bias" not in t else t["bias"].detach(), activation=activation,
                             residual=None if "residual" not in t else t["residual"].detach())]
    for leaf in _leaves(t):
        leaf.requires_grad_()
    y = fused_linear(t["x"], t["weight"], t.get("bias"), activation=activation, residual=t.get("residual"))
    return [y.detach(), *torch.autograd.grad(y, _leaves(t), t["dy"])]


def _check(t, activation, got):
    dtype = t["x"].dtype
    t = {k: v.detach().cpu() for k, v in t.items()}
    u, least, act_off = ROUNDOFF[dtype], SMALLEST[dtype], 2.0 ** -16 if dtype != torch.float32 else 2.0 ** -20
    x, w, dy = (t[k].double() for k in ("x", "weight", "dy"))
    bias = t["bias"].double() if "bias" in t else torch.zeros(w.shape[0], dtype=torch.float64)
    z = x @ w.T + bias
    ez = x.abs() @ w.abs().T * _sum(dtype, x.shape[1]) + U * (z.abs() + bias.abs())
    a, slope = _act(activation, z)

    def result(v, e, to):  # rounded once
        return e + (v.abs() + e) * ROUNDOFF[to] + SMALLEST[to]

    def near(g, want, bound, what):
        assert g.shape == want.shape, what
        g = g.double().cpu()
        worst = float(((g - want).abs() - bound).max()) if want.numel() else 0.0
        assert worst <= 0 and torch.isfinite(g).all(), (what, worst)

    # slopes are below 1.13, second derivatives below 1
    ea = 1.13 * ez + a.abs() * act_off
    y = a
    if "residual" in t:
        y = a + t["residual"].double()
        ea = ea + U * y.abs()
    y_type = t["residual"].dtype if "residual" in t else dtype
    assert got[0].dtype is y_type
    near(got[0], y, result(y, ea, y_type), "y")
    if len(got) == 1:
        return
    # z as it is kept, and its slope; where relu's corner is within reach it may be either
    kept = (z.abs() + ez) * u + least if activation is not None and dtype != torch.float32 else 0.0
    es = 0.0 if activation is None else (z.abs() <= ez).double() if activation == "relu" else ez + kept + (1 + slope.abs()) * act_off
    dz = dy * slope
    edz = dy.abs() * es + dz.abs() * 2 * U
    got = got[1:]
    db, edb = dz.sum(0), (edz + (dz.abs() + edz) * U * (64 + dz.shape[0] / 32)).sum(0)
    if dtype != torch.float32:
        edz = edz + (dz.abs() + edz) * u + least  # an operand

    def product(m, em, r):
        return m @ r, em @ r.abs() + (m.abs() + em) @ r.abs() * _sum(dtype, m.shape[1])

    for name, v, e in (("dx", *product(dz, edz, w)), ("dw", *product(dz.T, edz.T, x))):
        near(got[0], v, result(v, e, dtype), name)
        got = got[1:]
    if "bias" in t:
        near(got[0], db, result(db, edb, dtype), "db")
        got = got[1:]
    if "residual" in t:
        assert torch.equal(got[0].cpu(), t["dy"])


SIZES = [(1, 8, 8), (1, 64, 72), (3, 24, 40), (5, 1, 1), (7, 33, 1), (2, 1, 50), (33, 100, 60), (130, 264, 520), (257, 72, 1000), (300, 200, 731),
         (513, 64, 300), (100, 1024, 256), (70, 1000, 333), (300, 2048, 520)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("tokens,width,out", SIZES)
@pytest.mark.parametrize("dtype,activation,residual", [(torch.bfloat16, "gelu_tanh", None), (torch.float16, "gelu", torch.float16),
                                                       (torch.bfloat16, None, torch.float32), (torch.float32, "silu", torch.float32)])
def test_matches_64_bits(device, tokens, width, out, dtype, activation, residual):
    t = _inputs(tokens, width, out, dtype, residual, True, device)
    _check(t, activation, _call(t, activation))
    _check(t, activation, _call(t, activation, grad=False))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("residual", [None, "same", torch.float32])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("tokens,width,out", [(40, 72, 136), (9, 31, 45)])
def test_types_and_activations(device, dtype, activation, residual, bias, tokens, width, out):
    t = _inputs(tokens, width, out, dtype, dtype if residual == "same" else residual, bias, device, seed=1, scale=2.0)
    _check(t, activation, _call(t, activation))
    _check(t, activation, _call(t, activation, grad=False))


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 2, 7, 8, 9, 16, 17, 32, 33])
@pytest.mark.parametrize("width,out", [(512, 256), (1000, 2731), (264, 9480), (8, 9472), (33, 9500), (4096, 64)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_few_tokens(tokens, width, out, dtype):
    t = _inputs(tokens, width, out, dtype, dtype, True, "cuda", seed=tokens)
    _check(t, "gelu_tanh", _call(t, "gelu_tanh", grad=False))
    t = _inputs(tokens, width, out, dtype, torch.float32, False, "cuda", seed=tokens)
    _check(t, None, _call(t, None, grad=False))


@pytest.mark.gpu
def test_few_tokens_between_other_numbers():
    base = torch.full((40, 300), math.nan, device="cuda", dtype=torch.bfloat16)
    weights = torch.full((90, 301), math.nan, device="cuda", dtype=torch.bfloat16)
    out = torch.full((20, 90), math.nan, device="cuda", dtype=torch.bfloat16)
    for shift in range(0, 9):
        t = _inputs(5, 200, 77, torch.bfloat16, torch.bfloat16, True, "cuda", seed=shift)
        x, w, r = base[3:8, shift:shift + 200], weights[5:82, shift:shift + 200], out[2:7, shift:shift + 77]
        x.copy_(t["x"]), w.copy_(t["weight"]), r.copy_(t["residual"])
        t.update(x=x, weight=w, residual=r)
        _check(t, "silu", _call(t, "silu", grad=False))
        base.fill_(math.nan), weights.fill_(math.nan), out.fill_(math.nan)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,width,out,dtype,residual", [(2048, 1024, 1024, torch.bfloat16, torch.float32), (1500, 520, 4096, torch.float16, None),
                                                             (5000, 264, 2056, torch.bfloat16, torch.bfloat16), (1000, 1024, 1024, torch.float32, torch.float32)])
def test_many_tiles(tokens, width, out, dtype, residual):
    t = _inputs(tokens, width, out, dtype, residual, True, "cuda", seed=3)
    _check(t, "gelu", _call(t, "gelu"))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_one_of_the_gradients_alone(device, dtype):
    t = _inputs(40, 64, 72, dtype, torch.float32, True, device)
    full = _call(t, "gelu")[1:]
    for i, name in enumerate(("x", "weight", "bias", "residual")):
        for k in ("x", "weight", "bias", "residual"):
            t[k] = t[k].detach().requires_grad_(k == name)
        y = fused_linear(t["x"], t["weight"], t["bias"], activation="gelu", residual=t["residual"])
        (g,) = torch.autograd.grad(y, [t[name]], [t["dy"]])
        # (products side by side or alone add up alike here: no reduction is shared)
        assert torch.equal(g, full[i]), name


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_layouts(device, dtype):
    gen = torch.Generator().manual_seed(4)
    base = torch.randn(4, 6, 211, generator=gen).to(device, dtype)
    weight = torch.randn(90, 211, generator=gen).to(device, dtype)

    def both(x, w, r, dy, b):
        x, w, r, b = (v.detach().requires_grad_() for v in (x, w, r, b))
        y = fused_linear(x, w, b, activation="gelu", residual=r)
        return [y.detach(), *torch.autograd.grad(y, (x, w, r, b), dy)]

    for x in (base[..., :100], base[..., 1:101], base[..., 0:200:2], base.transpose(0, 1)[..., :100].transpose(0, 1), base[:1, :1, 4:104].expand(4, 6, 100)):
        for w in (weight[:, :100], weight[:, 3:103], weight[:, 0:200:2], weight.t()[:100].t(), weight[:1, :100].expand(90, 100)):
            r, dy, b = base[..., 7:97], base[..., 11:101], weight[:, 5]
            want = both(*(v.contiguous().clone() for v in (x, w, r, dy, b)))
            got = both(x, w, r, dy, b)
            # 100 terms of size one or so with other terms before or behind them
            assert all(torch.allclose(a.double(), c.double(), rtol=2 * ROUNDOFF[dtype], atol=200 * (U if dtype == torch.float32 else 2.0 ** -11) * 10) for a, c in zip(got, want))
    x = base[0, 0, :100]
    assert fused_linear(x, weight[:, :100]).shape == (90,)
    xs, w = base[..., :100].detach().requires_grad_(), weight[:, :100]
    g1 = torch.autograd.grad(fused_linear(xs, w, activation="relu").sum(), xs)[0]  # a gradient of stride zero
    g2 = torch.autograd.grad(fused_linear(xs, w, activation="relu"), xs, torch.ones(4, 6, 90, device=device, dtype=dtype))[0]
    assert torch.equal(g1, g2)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_infinities_nan_and_no_rows(device, dtype):
    x, w = torch.randn(6, 40, device=device).to(dtype), torch.randn(24, 40, device=device).to(dtype)
    x[1, 3], x[2, 5] = math.nan, math.inf
    for act in ACTIVATIONS:
        y = fused_linear(x, w, activation=act)
        assert torch.isnan(y[1]).all() and not torch.isfinite(y[2]).all() and torch.isfinite(y[[0, 3, 4, 5]]).all()
    for act in (None, "gelu"):
        t = {k: v.requires_grad_() for k, v in (("x", torch.zeros(0, 40, device=device, dtype=dtype)), ("w", w.clone()), ("b", torch.zeros(24, device=device, dtype=dtype)))}
        y = fused_linear(t["x"], t["w"], t["b"], activation=act)
        gx, gw, gb = torch.autograd.grad(y.sum(), list(t.values()))
        assert y.shape == (0, 24) and gx.shape == (0, 40) and float(gw.abs().sum()) == 0 and float(gb.abs().sum()) == 0 and gb.shape == (24,)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("activation", ["relu", "silu", "gelu", "gelu_tanh"])
def test_far_out(device, dtype, activation):
    # one weight of one: z is x.  Slopes are 0 and 1 far out, also where z is beyond fp16's range.
    ends = [-6e4, -300.0, -88.0, -30.0, 30.0, 88.0, 300.0, 6e4]
    x = torch.tensor(ends, device=device).to(dtype)[:, None].requires_grad_()
    w = torch.ones(1, 1, device=device, dtype=dtype)
    b = torch.zeros(1, device=device, dtype=dtype)
    y = fused_linear(x, w, b, activation=activation)
    (g,) = torch.autograd.grad(y, x, torch.ones_like(y))
    # (silu's slope at -30 is 29 exp(-30), 2.8e-12, below zero)
    assert ((g[:, 0].float().cpu() - torch.tensor([0.0] * 4 + [1.0] * 4)).abs() <= 3e-12).all() and torch.equal(y[4:], x.detach()[4:]) and (y[:4].float().abs() < 1e-10).all()
    x = torch.full((3, 2), 5e4, device=device).to(dtype).requires_grad_()
    y = fused_linear(x, torch.ones(1, 2, device=device, dtype=dtype), activation=activation, residual=torch.zeros(3, 1, device=device))
    assert torch.equal(torch.autograd.grad(y, x, torch.ones_like(y))[0], torch.ones_like(x))
    assert (y == 2 * x.detach()[:, :1].float()).all()


@pytest.mark.parametrize("device", DEVICES)
def test_gradients_are_those_of_differences(device):
    t = _inputs(6, 30, 20, torch.float32, torch.float32, True, device, seed=5)
    gen = torch.Generator().manual_seed(8)
    for activation in ("silu", "gelu", "gelu_tanh", None):
        grads = _call(t, activation)[1:]
        for name, grad in zip(("x", "weight", "bias", "residual"), grads):
            way = torch.randn(t[name].shape, generator=gen).to(device)
            h = 2.0 ** -8

            def value(sign):
                moved = {k: v.detach() for k, v in t.items()}
                moved[name] = moved[name] + sign * h * way
                return float((_call(moved, activation, grad=False)[0].double() * t["dy"].double()).sum())

            got, want = (value(1) - value(-1)) / (2 * h), float((grad.double() * way.double()).sum())
            # 120 results, each off by some 50 roundings of its size of a few, over h; third derivatives (below 2) of steps of up to
            # 5 h each, cubed and weighted with dy
            assert abs(got - want) <= 120 * 4 * 50 * U / h + 120 * 2 * 125 * h * h / 6


@pytest.mark.parametrize("device", DEVICES)
def test_module_autocast_and_modes(device):
    torch.manual_seed(2)
    m = FusedLinear(48, 40, activation="gelu").to(device)
    ref = torch.nn.Linear(48, 40).to(device)
    ref.load_state_dict(m.state_dict())
    m.requires_grad_(False), ref.requires_grad_(False)
    x, other, r = torch.randn(7, 48, device=device), torch.randn(7, 48, device=device), torch.randn(7, 40, device=device)
    assert torch.allclose(m(x, r), torch.nn.functional.gelu(ref(x)) + r, rtol=0, atol=1e-5)
    with torch.autocast(device, dtype=torch.bfloat16):
        y, y32 = m(x), m(x, r)
    assert y.dtype is torch.bfloat16 and y32.dtype is torch.float32
    lone = [t.bfloat16() for t in (x, m.weight, m.bias)]
    assert torch.equal(y, fused_linear(*lone, activation="gelu")) and torch.equal(y32, fused_linear(*lone, activation="gelu", residual=r))
    w = m.weight.clone().requires_grad_()
    with torch.autocast(device, dtype=torch.bfloat16):
        z = fused_linear(x, w, m.bias, activation="silu")
        (g,) = torch.autograd.grad(z, w, torch.ones_like(z))
    assert g.dtype is torch.float32
    for pre in (False, True):
        traced = make_fx(lambda t: fused_linear(t, m.weight, m.bias, activation="gelu"), pre_dispatch=pre)(x)
        assert torch.allclose(traced(other), m(other), rtol=0, atol=1e-5)
    with FlopCounterMode(display=False) as count:
        y = fused_linear(x.requires_grad_(), w, m.bias, activation="gelu")
        torch.autograd.grad(y, (x, w), torch.ones_like(y))
    assert count.get_total_flops() == 3 * 2 * 7 * 48 * 40


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    x, w, b = torch.randn(4, 16, device=device).half(), torch.randn(24, 16, device=device).half(), torch.randn(24, device=device).half()
    kind = ValueError if device == "cpu" else RuntimeError
    r = torch.randn(4, 24, device=device)
    for args, kw in [((x.float(), w), {}), ((x, w, b.float()), {}), ((x, w[:, :8]), {}), ((x, w, b[:8]), {}), ((x, w[0]), {}), ((x, w[:0]), {}), ((x[:, :0], w[:, :0]), {}),
                     ((x[0, 0], w), {}), ((x, w, b[None]), {}), ((x, w), dict(residual=r[:2])), ((x, w), dict(residual=r.bfloat16())), ((x, w), dict(residual=r[:, :1])),
                     ((x, w), dict(residual=r.double()))]:
        with pytest.raises(kind, match="fused_linear"):
            fused_linear(*args, **kw)
    for bad in ("tanh", "none", "GELU"):
        with pytest.raises(ValueError, match="activation"):
            fused_linear(x, w, activation=bad)
    with pytest.raises(ValueError, match="activation"):
        FusedLinear(4, 4, activation="tanh")


@pytest.mark.gpu
def test_refusals_of_the_kernels(cuda_device):
    x, w = torch.randn(4, 16, device=cuda_device, requires_grad=True), torch.randn(24, 16, device=cuda_device)
    with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
        fused_linear(x.double(), w.double())
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        fused_linear(x, w.cpu())
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(fused_linear(x, w, activation="gelu").sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="fused_linear"):
        torch.func.vmap(lambda t: fused_linear(t[None], w))(x.detach())
    y = fused_linear(x, w)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(lambda t: torch.autograd.grad(y, x, t, retain_graph=True)[0])(torch.ones_like(y))
    for change in (lambda t: t.double(), lambda t: t[:2], lambda t: t.cpu()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
            y = fused_linear(x, w, activation="relu")
        with pytest.raises(RuntimeError, match="fused_linear: a (tensor saved for the backward pass|dense CUDA tensor)"):
            torch.autograd.grad(y, x, torch.ones_like(y))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_saved_tensors_that_come_back_laid_out_anew(cuda_device, dtype):
    t = _inputs(70, 40, 56, dtype, None, True, cuda_device)
    want = _call(t, "gelu")
    for hooks in ((lambda v: v, lambda v: v.t().contiguous().t() if v.dim() == 2 else v), (lambda v: v.cpu(), lambda v: v.to(cuda_device))):
        with torch.autograd.graph.saved_tensors_hooks(*hooks):
            y = fused_linear(*_leaves(t), activation="gelu")
        got = [y.detach(), *torch.autograd.grad(y, _leaves(t), t["dy"])]
        assert all(torch.allclose(a.double(), b.double(), rtol=2 * ROUNDOFF[dtype], atol=1e-4) for a, b in zip(got, want))


@pytest.mark.gpu
def test_results_do_not_depend_on_the_run(cuda_device):
    t = _inputs(3000, 264, 1032, torch.bfloat16, torch.float32, True, cuda_device)
    first = _call(t, "gelu_tanh")
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, _call(t, "gelu_tanh")))


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [3, 200])
def test_captured_replayed_and_on_another_stream(cuda_device, tokens):
    t = _inputs(tokens, 200, 136, torch.bfloat16, torch.float32, True, cuda_device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            out = _call(t, "gelu")
            few = _call(t, "gelu", grad=False)
    torch.cuda.current_stream().wait_stream(side)
    _check(t, "gelu", out), _check(t, "gelu", few)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _call(t, "gelu")
        few = _call(t, "gelu", grad=False)
    other = _inputs(tokens, 200, 136, torch.bfloat16, torch.float32, True, cuda_device, seed=8)
    with torch.no_grad():
        for k, v in other.items():
            t[k].copy_(v)
    graph.replay()
    _check(t, "gelu", out), _check(t, "gelu", few)


@pytest.mark.gpu
def test_waits_that_run_out_are_reported_and_leave_nan():
    # in a process of its own: the report is one for the whole device
    code = """
import torch, mccl_b200
from mccl_b200.ops.fused_linear import fused_linear
native = mccl_b200.require_native()
x, w = (torch.randn(*s, device="cuda").bfloat16() for s in ((300, 256), (512, 256)))
y = native._fused_linear_with_limit(x, w, 0)
torch.cuda.synchronize()
assert torch.isnan(y).all()
try:
    fused_linear(x, w)
except RuntimeError as e:
    assert "ran out" in str(e)
else:
    raise AssertionError("not reported")
assert torch.isfinite(fused_linear(x, w)).all()
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.fixture
def emptied():
    """What a test of several GB leaves in torch's cache is given back behind it: other tests count on what is free."""
    yield
    torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("activation,residual", [("gelu", None), (None, torch.float32)])
def test_places_beyond_32_bits(emptied, cuda_device, activation, residual):
    tokens, out, width = 70000, 32776, 24
    gen = torch.Generator(device=cuda_device).manual_seed(2)
    x, w = (torch.randn(*s, generator=gen, device=cuda_device).bfloat16() for s in ((tokens, width), (out, width)))
    r = None
    if residual is not None:
        r = torch.empty(tokens, out, device=cuda_device, dtype=residual).normal_(generator=gen)
    x.requires_grad_()
    y = fused_linear(x, w, activation=activation, residual=r)
    ends = torch.tensor([0, 1, 65535, 65536, tokens - 2, tokens - 1], device=cuda_device)
    part = x.detach()[ends].requires_grad_()
    want = fused_linear(part, w, activation=activation, residual=None if r is None else r[ends])
    # (few tokens that keep nothing have a kernel of their own, with another order of the sums)
    size = x.detach()[ends].abs().double() @ w.abs().double().T
    off = (y.detach()[ends].double() - want.detach().double()).abs()
    assert (off == 0).all() if residual is None else (off <= 2 * _sum(torch.bfloat16, width) * size + 2 * U * want.detach().abs().double()).all()
    dy = y.detach()
    (g,) = torch.autograd.grad(y, x, dy)
    (few,) = torch.autograd.grad(want, part, dy[ends])
    # (a sum of 32776 terms whose order and parts may differ)
    size = dy[ends].abs().double() @ w.abs().double()
    assert ((g[ends].double() - few.double()).abs() <= few.abs().double() * 2.0 ** -7 + size * (out / 8 + 40) * 2.0 ** -22).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_one_tensor_twice(device, dtype):
    # x beside itself as the residual, and a matrix times itself
    t = _inputs(40, 40, 40, dtype, dtype, True, "cpu")

    def run(x, to):
        y = to(x)
        y.backward(t["dy"].to(y.device, y.dtype))
        return y.detach().double().cpu(), x.grad.double().cpu()

    bias = t["bias"].to(device)
    for of, plain in ((lambda x: fused_linear(x, x, bias, residual=x), lambda x: x @ x.t() + t["bias"].double() + x),
                      (lambda x: fused_linear(x.t(), x, residual=x), lambda x: x.t() @ x.t() + x)):
        got = run(t["x"].to(device, copy=True).requires_grad_(), of)
        want = run(t["x"].double().requires_grad_(), plain)
        for a, b in zip(got, want):
            # 3 gradients of one leaf, each rounded, and their two sums: 5 half steps of at most the sum of their sizes, some 4 of the largest entry
            assert (a - b).abs().max() <= 20 * ROUNDOFF[dtype] * b.abs().max()


@pytest.mark.gpu
@pytest.mark.parametrize("activation", [None, "gelu"])
@pytest.mark.parametrize("tokens,width,out", [(1, 1, 1), (31, 33, 65), (1024, 64, 512), (1025, 64, 512), (1000, 128, 513), (8192, 5, 7), (8200, 5, 7), (64, 257, 130), (700, 77, 176),
                                              (2, 256, 8192), (3, 5000, 100)])
def test_small_in_full_precision(cuda_device, tokens, width, out, activation):
    # either side of where products are the library's, and sums in both directions over parts of a stage
    t = _inputs(tokens, width, out, torch.float32, torch.float32, True, cuda_device)
    _check(t, activation, _call(t, activation))
    t = {k: v.detach() for k, v in t.items()}
    for k in ("x", "weight", "residual", "dy"):  # rows that lie apart
        t[k] = torch.cat((t[k], torch.full_like(t[k], math.nan)), 1)[:, :t[k].shape[1]]
    t["bias"] = torch.stack((t["bias"], t["bias"]), 1)[:, 0]
    _check(t, activation, _call(t, activation))


@pytest.mark.gpu
def test_small_in_full_precision_one_gradient_alone(cuda_device):
    t = _inputs(50, 40, 60, torch.float32, None, True, cuda_device)
    whole = _call(t, None)[1:]
    for i, leaf in enumerate(_leaves(t)):
        others = {k: v.detach() for k, v in t.items()}
        name = ("x", "weight", "bias")[i]
        others[name].requires_grad_()
        y = fused_linear(others["x"], others["weight"], others["bias"])
        assert torch.equal(torch.autograd.grad(y, others[name], t["dy"])[0], whole[i])


@pytest.mark.gpu
def test_two_threads_on_streams_of_their_own(cuda_device):
    from concurrent.futures import ThreadPoolExecutor
    cases = [_inputs(tokens, 264, out, torch.bfloat16, torch.float32, True, cuda_device, seed=out) for tokens, out in ((9, 136), (333, 1032), (3000, 1032), (3000, 520))]
    want = [_call(t, "gelu") for t in cases]
    torch.cuda.synchronize()

    def many(t):
        with torch.cuda.stream(torch.cuda.Stream()):
            got = [_call(t, "gelu") for _ in range(8)]
            torch.cuda.current_stream().synchronize()
        return got

    with ThreadPoolExecutor(len(cases)) as pool:
        for got, one in zip(pool.map(many, cases), want):
            assert all(torch.equal(a, b) for g in got for a, b in zip(g, one))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype,activation", [(torch.float32, None), (torch.float32, "gelu"), (torch.bfloat16, None), (torch.bfloat16, "gelu")])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("shape", [(24,), (6, 24), (2, 3, 24), (2, 3, 4, 24)])
def test_gradients_of_leaves_have_memory_of_their_own(device, dtype, activation, wide, shape):
    gen = torch.Generator().manual_seed(4)
    kind = torch.float32 if wide else dtype
    x, r, w = (torch.randn(s, generator=gen).to(device, t).requires_grad_() for s, t in ((shape, dtype), (shape, kind), ((24, 24), dtype)))
    given = torch.randn(shape, generator=gen).to(device, kind)
    kept = given.clone()
    for turn in (1, 2):
        y = fused_linear(x, w, activation=activation, residual=r)
        one = torch.autograd.grad(y, (x, w, r), given, retain_graph=True)
        y.backward(given)
        # (the same numbers twice are twice these, exactly)
        assert y.shape == shape and all(torch.equal(t.grad, turn * g) for t, g in zip((x, w, r), one))
        assert len({t.untyped_storage().data_ptr() for t in (x.grad, w.grad, r.grad, given)}) == 4
    assert torch.equal(given, kept)


@pytest.fixture
def emptied():
    yield
    torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("width,out", [(64, 64), (61, 300)])
def test_long_sums_that_are_shared_too(emptied, cuda_device, width, out):
    # one tile or two, whose reduction 16 pairs share, each with more than 2^15 terms
    gen = torch.Generator(device=cuda_device).manual_seed(out)
    x = torch.rand(600_001, width, device=cuda_device, generator=gen, dtype=torch.float16)
    w = torch.rand(out, width, device=cuda_device, generator=gen, dtype=torch.float16).requires_grad_()
    dy = torch.rand(600_001, out, device=cuda_device, generator=gen, dtype=torch.float16) * 2.0 ** -10
    before = _launches()
    (got,) = torch.autograd.grad(fused_linear(x, w), w, dy)
    assert _launches() >= before + 3
    want = dy.double().t() @ x.double()
    assert ((got.double() - want).abs() / want).max() <= 68 * 2.0 ** -23 + (600_001 / 512 / 16 + 17) * U + ROUNDOFF[torch.float16] * 1.01


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,tokens", [(torch.float16, 32768), (torch.float16, 32769), (torch.float16, 262144), (torch.bfloat16, 262144), (torch.bfloat16, 262145)])
@pytest.mark.parametrize("both", [False, True])
@pytest.mark.parametrize("width", [2048, 2043])
def test_weight_gradients_of_many_tokens_of_one_sign(emptied, cuda_device, dtype, tokens, both, width):
    gen = torch.Generator(device=cuda_device).manual_seed(tokens)
    x = torch.rand(tokens, width, device=cuda_device, generator=gen, dtype=dtype).requires_grad_(both)
    w = torch.rand(2048, width, device=cuda_device, generator=gen, dtype=dtype).requires_grad_()
    # 64 terms of the sums are of size one
    dy = torch.rand(tokens, 2048, device=cuda_device, generator=gen, dtype=dtype) * (64.0 / tokens)
    got = torch.autograd.grad(fused_linear(x, w), (x, w) if both else w, dy)
    rows, columns = (torch.arange(0, n, 7, device=cuda_device) for n in (2048, width))
    want = dy[:, rows].double().t() @ x.detach()[:, columns].double()
    # Sums of up to 2^15 terms (bf16 2^18): each 8 of them cut off at 2^-23.  Longer ones: 512 terms so, added up in fp32.  The result is rounded once.
    longest = 1 << (15 if dtype is torch.float16 else 18)
    off = ((got[-1][rows][:, columns].double() - want).abs() / want).max()
    assert off <= ((tokens / 8 + 4) * 2.0 ** -23 if tokens <= longest else 68 * 2.0 ** -23 + tokens / 512 * U) + ROUNDOFF[dtype] * 1.01
    if both:
        rows = torch.arange(0, tokens, tokens // 97, device=cuda_device)
        want = dy[rows].double() @ w.detach().double()
        assert ((got[0][rows].double() - want).abs() / want).max() <= _sum(dtype, 2048) + ROUNDOFF[dtype] * 1.01


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype,residual", [(torch.float32, None), (torch.float16, None), (torch.bfloat16, None), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("tokens,out", [(3, 24), (40, 45), (700, 64)])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_relu_leaves_nothing_of_a_gradient_that_is_not_finite_below_zero(device, dtype, residual, tokens, out, value):
    t = _inputs(tokens, 16, out, dtype, residual, True, device, seed=6)
    z = (t["x"].double() @ t["weight"].double().t() + t["bias"].double()).cpu()
    low, high = (z < -0.1).nonzero()[0].tolist(), (z > 0.1).nonzero()[-1].tolist()
    clean = t["dy"].clone()
    clean[low[0], low[1]] = 0
    t["dy"][low[0], low[1]] = value
    got = _call(t, "relu")[1:]
    want = _call({**t, "dy": clean}, "relu")[1:]
    for a, b in list(zip(got, want))[:3]:  # the residual's gradient is dy itself
        assert torch.isfinite(a).all() and torch.equal(a, b)
    # above zero it goes on, as where z is a NaN
    t["dy"] = clean.clone()
    t["dy"][high[0], high[1]] = value
    got = _call(t, "relu")[1:]
    assert not torch.isfinite(got[0][high[0]]).any() and not torch.isfinite(got[1][high[1]]).any() and not torch.isfinite(got[2][high[1]])
    x = torch.full((2, 16), math.nan, device=device, dtype=dtype).requires_grad_()
    y = fused_linear(x, t["weight"].detach(), activation="relu")
    assert torch.equal(torch.autograd.grad(y, x, torch.ones_like(y))[0], torch.autograd.grad(fused_linear(x, t["weight"].detach()), x, torch.ones_like(y))[0])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_result_that_nobody_has_a_gradient_of(device, dtype):
    class Stop(torch.autograd.Function):
        @staticmethod
        def forward(ctx, y):
            return y.clone()

        @staticmethod
        def backward(ctx, dy):
            return None

    t = _inputs(9, 24, 40, dtype, dtype, True, device)
    leaves = [v.requires_grad_() for v in _leaves(t)]
    y = fused_linear(t["x"], t["weight"], t["bias"], activation="gelu", residual=t["residual"])
    assert torch.autograd.grad(Stop.apply(y).sum(), leaves, allow_unused=True) == (None,) * 4


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("tokens,width,out", [(3, 24, 40), (300, 72, 1000), (256, 1024, 520)])
def test_nothing_is_kept_for_the_residuals_gradient(device, dtype, tokens, width, out):
    t = _inputs(tokens, width, out, dtype, torch.float32, True, device, seed=2)
    t["residual"].requires_grad_()
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda s: kept.append(s.shape) or s, lambda s: s):
        y = fused_linear(t["x"], t["weight"], t["bias"], activation="gelu", residual=t["residual"])
    # the operands, which are the caller's
    assert all(tuple(s) in ((tokens, width), (out, width)) for s in kept)
    assert torch.equal(torch.autograd.grad(y, t["residual"], t["dy"])[0], t["dy"])
    for name in ("x", "weight", "bias"):  # one other is enough
        u = {k: v.detach().requires_grad_(k in (name, "residual")) for k, v in t.items()}
        full = {k: v.detach().requires_grad_(k != "dy") for k, v in t.items()}
        a, b = (fused_linear(v["x"], v["weight"], v["bias"], activation="gelu", residual=v["residual"]) for v in (u, full))
        # (few tokens of which nothing is kept have a kernel of their own)
        assert torch.equal(torch.autograd.grad(a, u[name], t["dy"])[0], torch.autograd.grad(b, full[name], t["dy"])[0])


def _launches():
    from mccl_b200 import require_native
    return require_native()._kernel_launches()


@pytest.mark.gpu
@pytest.mark.parametrize("out", [1504, 1503])
@pytest.mark.parametrize("dtype,residual", [(torch.float16, None), (torch.bfloat16, None), (torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16),
                                            (torch.float16, torch.float32), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("activation", [None, "gelu"])
def test_tiles_whose_reduction_is_shared(cuda_device, out, dtype, residual, activation):
    # 13 x 6 tiles of 256 x 256 for 74 pairs: the last four are shared, and a second launch adds their parts up
    t = _inputs(3300, 1024, out, dtype, residual, True, cuda_device, seed=out)
    before = _launches()
    y = _call(t, activation, grad=False)
    assert _launches() == before + 2
    _check(t, activation, y)
    _check(t, activation, _call(t, activation))


@pytest.mark.gpu
@pytest.mark.parametrize("out", [3000, 3001])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("residual", [None, torch.float32])
@pytest.mark.parametrize("activation", [None, "gelu_tanh"])
def test_several_tiles_a_pair_of_several_parts_each(cuda_device, out, dtype, residual, activation):
    # 25 x 12 tiles for 74 pairs, four whole ones each and four that are shared; sums of 1600 leave tensor memory in four parts where y is in 32 bits
    t = _inputs(6400, 1600, out, dtype, residual, True, cuda_device, seed=out)
    rows = torch.arange(0, 6400, 37, device=cuda_device)
    some = {k: v[rows] if k in ("x", "residual", "dy") else v for k, v in t.items()}
    before = _launches()
    y = _call(t, activation, grad=False)[0]
    assert _launches() == before + 2
    _check(some, activation, [y[rows]])
    saved = []
    t["x"].requires_grad_()
    with torch.autograd.graph.saved_tensors_hooks(lambda s: saved.append(s) or s, lambda s: s):
        kept = fused_linear(t["x"], t["weight"], t["bias"], activation=activation, residual=t.get("residual"))
    assert torch.equal(kept, y)
    if activation is None:
        return
    (z,) = (s for s in saved if s.shape == (6400, (out + 7) // 8 * 8))
    x, w, b = (some[k].detach().double() for k in ("x", "weight", "bias"))
    want = x @ w.T + b
    ez = x.abs() @ w.abs().T * _sum(dtype, 1600) + U * (want.abs() + b.abs())
    assert ((z[rows, :out].double() - want).abs() <= ez + (want.abs() + ez) * ROUNDOFF[dtype] + SMALLEST[dtype]).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("shape", [(16,), (5, 16), (2, 3, 16), (2, 2, 3, 16)])
def test_tensors_that_are_changed_in_place(device, shape):
    w = torch.randn(16, 16, device=device, requires_grad=True)
    for activation in (None, "gelu"):
        x = torch.randn(shape, device=device, requires_grad=True) * 2
        y = fused_linear(x, w, activation=activation, residual=x)
        x.add_(1)  # what backward would read
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
        x = torch.randn(shape, device=device, requires_grad=True) * 2
        y = fused_linear(x, w, activation=activation, residual=x)
        y.mul_(2)  # what it would not
        y.sum().backward()
