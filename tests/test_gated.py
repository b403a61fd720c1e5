"""The gated feed-forward block against its formulas in 64 bits."""
import math
import subprocess
import sys
import threading
from pathlib import Path

import pytest
import torch

import mccl_b200
from mccl_b200.ops.checkpoint import GROUP, pack8, unpack8
from mccl_b200.ops.gated import GatedFeedForward, gated_feed_forward

ROUNDOFF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def _act(name, z):
    c = 2 * math.sqrt(2 / math.pi)
    s = torch.sigmoid(z if name == "silu" else c * (z + 0.044715 * z ** 3))
    return z * s, s + z * s * (1 - s) * (1 if name == "silu" else c * (1 + 3 * 0.044715 * z * z))


class Rounding:
    """What each step may add to the error, for a type.

    Products of 16-bit numbers are exact in fp32; the tensor cores cut each sum of (at least) 8 of them off at 2^-23 of what it
    adds up.  fp32 products are six bf16 products (2^-20, see the linear layer's test) or sums of a library kernel (2^-24 a term).
    """
    def __init__(self, dtype):
        self.dtype, self.half = dtype, dtype != torch.float32
        self.out, self.least = ROUNDOFF[dtype], SMALLEST[dtype]
        # the logistic function: an exponential within (2 + 1.2 |z|) 2^-23 of its own, |z| below 100, and a quotient
        self.act = 2.0 ** -16 if self.half else 2.0 ** -20
        self.keep = 2.0 ** -16 if self.half else 0.0

    def sum(self, depth):
        return (depth / 8 + 4) * 2.0 ** -23 if self.half else 2.0 ** -20 + (depth + 2) * 2.0 ** -24

    def mid(self, v):  # h, dg, du as operands
        return v.abs() * self.out + self.least if self.half else v.abs() * 2.0 ** -23

    def result(self, v, e):
        return e + (v.abs() + e) * self.out + self.least


def _keep8(v, e):
    """Values kept in 8 bits of exact ones that the kernel has within e, and how far its own may be: a code may be the next one
    where the exact value is that near to the middle of two."""
    out, err = torch.empty_like(v), torch.empty_like(v)
    for at in range(0, v.shape[1], GROUP):
        g, eg = v[:, at:at + GROUP], e[:, at:at + GROUP]
        most = g.abs().amax(1, keepdim=True)
        scale = most / 127
        safe = torch.where(scale > 0, scale, 1.0)
        t = g / safe
        code = torch.round(t)
        e_scale = eg.amax(1, keepdim=True) / 127 + scale * 2.0 ** -23
        slack = eg / safe + 128 * (e_scale / safe + 2.0 ** -22)
        flips = ((t - torch.floor(t)) - 0.5).abs() <= slack
        out[:, at:at + GROUP] = code * scale
        err[:, at:at + GROUP] = code.abs() * e_scale + flips * (scale + e_scale)
    return out, err


def _want(x, wg, wu, wd, dy, name, eight, r):
    """{result: (value, bound)} in 64 bits."""
    x, wg, wu, wd = (t.detach().double() for t in (x, wg, wu, wd))
    width, hidden, tokens = x.shape[1], wg.shape[0], x.shape[0]
    g, u = x @ wg.T, x @ wu.T
    eg, eu = (x.abs() @ w.abs().T * r.sum(width) for w in (wg, wu))
    a, _ = _act(name, g)
    h = a * u
    # the slopes of both activations are below 1.13, their second derivatives below 1
    eh = 1.13 * eg * u.abs() + (a.abs() + 1.13 * eg) * eu + h.abs() * r.act
    eh = eh + r.mid(h.abs() + eh)
    y = h @ wd.T
    got = {"y": (y, r.result(y, eh @ wd.abs().T + (h.abs() + eh) @ wd.abs().T * r.sum(hidden)))}
    if dy is None:
        return got
    dy = dy.double()
    if eight:
        x = unpack8(pack8(x.to(r.dtype))).double()  # bit for bit: see the checkpoints' own test
        (g, eg), (u, eu) = _keep8(g, eg), _keep8(u, eu)
    else:
        eg, eu = eg + r.keep * (g.abs() + eg), eu + r.keep * (u.abs() + eu)
    a, slope = _act(name, g)
    ea, es = 1.13 * eg + a.abs() * r.act, eg + (1 + slope.abs()) * r.act
    dh = dy @ wd
    edh = dy.abs() @ wd.abs() * r.sum(width)

    def product(*factors):  # and its error
        value, total, clean = 1.0, 1.0, 1.0
        for f, e in factors:
            value, total, clean = value * f, total * (f.abs() + e), clean * f.abs()
        e = total - clean + clean * 2.0 ** -22
        return value, e + r.mid(value.abs() + e)

    h, eh = product((a, ea), (u, eu))
    dg, edg = product((dh, edh), (u, eu), (slope, es))
    du, edu = product((dh, edh), (a, ea))

    def times(left, right):  # sum over the last of the left, first of the right
        (m, em), w = left, right.abs()
        return m @ right, em @ w + (m.abs() + em) @ w * r.sum(m.shape[1])

    (p, ep), (q, eq) = times((dg, edg), wg), times((du, edu), wu)
    dx, edx = p + q, ep + eq + ((dg.abs() + edg) @ wg.abs() + (du.abs() + edu) @ wu.abs()) * (r.sum(hidden) + 2.0 ** -23)
    got["dx"] = (dx, r.result(dx, edx))
    for key, left in (("dw_gate", (dg.T, edg.T)), ("dw_up", (du.T, edu.T))):
        v, e = times(left, x)
        got[key] = (v, r.result(v, e))
    v, e = times((h.T, eh.T), dy)
    got["dw_down"] = (v.T, r.result(v, e).T)
    return got


def _inputs(tokens, width, hidden, dtype, seed=0, device="cuda"):
    gen = torch.Generator(device=device).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen, device=device)  # noqa: E731
    return (rand(tokens, width).to(dtype), (rand(hidden, width) * width ** -0.5).to(dtype), (rand(hidden, width) * width ** -0.5).to(dtype),
            (rand(width, hidden) * hidden ** -0.5).to(dtype), rand(tokens, width).to(dtype))


def _check(got, want):
    for key, (value, bound) in want.items():
        g = got[key].detach().double()
        assert g.shape == value.shape, key
        off = (g - value).abs() - bound
        assert (off <= 0).all(), (key, off.max().item(), bound.max().item())


def _pass(args, dy, **kw):
    y = gated_feed_forward(*args, **kw)
    return dict(zip(("y", "dx", "dw_gate", "dw_up", "dw_down"), (y, *torch.autograd.grad(y, args, dy))))


# one token and a few; tiles and groups that end inside; widths that are no multiple of 16 bytes; shared and whole reductions
SIZES = [
    (1, 64, 64), (1, 1024, 2816), (2, 8, 8), (3, 1, 1), (5, 127, 65), (17, 200, 328), (64, 512, 1024), (100, 96, 130), (128, 128, 128), (129, 130, 257),
    (256, 1000, 2731), (333, 264, 520), (700, 328, 200), (1025, 136, 392), (2100, 64, 72), (40, 2048, 136), (40, 136, 4096),
]


@pytest.mark.gpu
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("dtype,activation", [(torch.bfloat16, "silu"), (torch.float16, "gelu_tanh"), (torch.float32, "silu"), (torch.float32, "gelu_tanh")])
@pytest.mark.parametrize("tokens,width,hidden", SIZES)
def test_matches_64_bits(tokens, width, hidden, dtype, activation, eight):
    *args, dy = _inputs(tokens, width, hidden, dtype, seed=tokens + width)
    want = _want(*args, dy, activation, eight, Rounding(dtype))
    args = [t.requires_grad_() for t in args]
    got = _pass(args, dy, activation=activation, checkpoint="int8" if eight else None)
    _check(got, want)
    with torch.no_grad():
        _check({"y": gated_feed_forward(*args, activation=activation)}, {"y": want["y"]})


# single tokens and a few: their own kernels, at whole and ragged rows
@pytest.mark.gpu
@pytest.mark.parametrize("dtype,activation", [(torch.bfloat16, "silu"), (torch.float16, "gelu_tanh")])
@pytest.mark.parametrize("width,hidden", [(1024, 2816), (1000, 2731), (8, 24), (5, 3), (256, 264), (3000, 520), (136, 9000)])
@pytest.mark.parametrize("tokens", [1, 2, 3, 4, 7, 8, 9, 16, 17, 25, 32, 33])
def test_few_tokens_match_64_bits(tokens, width, hidden, dtype, activation):
    x, wg, wu, wd, _ = _inputs(tokens, width, hidden, dtype, seed=tokens)
    want = _want(x, wg, wu, wd, None, activation, False, Rounding(dtype))
    _check({"y": gated_feed_forward(x, wg, wu, wd, activation=activation)}, want)

    def odd(t):
        big = torch.zeros(t.shape[0], t.shape[1] + 5, dtype=dtype, device="cuda")[:, 3:3 + t.shape[1]]
        return big.copy_(t)

    _check({"y": gated_feed_forward(odd(x), odd(wg), wu.t().contiguous().t(), odd(wd), activation=activation)}, want)
    same = gated_feed_forward(x[:1].expand(tokens, width), wg, wu, wd, activation=activation)
    _check({"y": same[-1:]}, {"y": tuple(t[:1] for t in want["y"])})


# on both sides of the sizes at which a few tokens of wide blocks become tiles
@pytest.mark.gpu
@pytest.mark.parametrize("tokens,width,hidden", [(1, 7168, 7000), (2, 7168, 7048), (3, 4096, 8100), (8, 4096, 8209), (16, 2048, 4096), (9, 2048, 4104),
                                                 (32, 1024, 4096), (17, 1000, 4211)])
def test_few_tokens_of_wide_blocks_match_64_bits(tokens, width, hidden):
    x, wg, wu, wd, _ = _inputs(tokens, width, hidden, torch.bfloat16, seed=tokens)
    _check({"y": gated_feed_forward(x, wg, wu, wd)}, _want(x, wg, wu, wd, None, "silu", False, Rounding(torch.bfloat16)))


@pytest.mark.gpu
@pytest.mark.parametrize("activation", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("width,hidden", [(1024, 2816), (1000, 2731), (999, 514), (8, 24), (5, 3), (1, 1), (260, 136), (136, 9000), (3000, 1500)])
@pytest.mark.parametrize("tokens", [1, 2, 3, 4, 5, 8, 9, 13, 16, 17])
def test_few_tokens_of_float32_match_64_bits(tokens, width, hidden, activation):
    x, wg, wu, wd, _ = _inputs(tokens, width, hidden, torch.float32, seed=tokens)
    want = _want(x, wg, wu, wd, None, activation, False, Rounding(torch.float32))
    _check({"y": gated_feed_forward(x, wg, wu, wd, activation=activation)}, want)

    def among(t, shift):
        big = torch.full((t.shape[0] + 2, t.shape[1] + 5 + shift), float("nan"), device="cuda")
        return big[1:-1, shift:shift + t.shape[1]].copy_(t)

    for shift in range(4):
        _check({"y": gated_feed_forward(among(x, shift), among(wg, 3 - shift), wu.t().contiguous().t(), among(wd, shift), activation=activation)}, want)
    same = gated_feed_forward(x[:1].expand(tokens, width), wg, wu, wd, activation=activation)
    _check({"y": same[-1:]}, {"y": tuple(t[:1] for t in want["y"])})
    bad = x.clone()
    bad[0, width // 2] = float("nan")
    got = gated_feed_forward(bad, wg, wu, wd, activation=activation)
    assert torch.isnan(got[0]).all() and torch.isfinite(got[1:]).all()


# rows at every distance from 16 bytes, among numbers that are not theirs
@pytest.mark.gpu
@pytest.mark.parametrize("tokens,width,hidden", [(1, 1023, 515), (3, 70, 33), (8, 517, 1030), (13, 259, 771), (30, 333, 130)])
@pytest.mark.parametrize("shift", range(8))
def test_few_tokens_between_other_numbers(tokens, width, hidden, shift):
    x, wg, wu, wd, _ = _inputs(tokens, width, hidden, torch.float16, seed=shift)
    want = _want(x, wg, wu, wd, None, "silu", False, Rounding(torch.float16))

    def among(t, pad):
        big = torch.full((t.shape[0] + 2, t.shape[1] + shift + pad), float("nan"), dtype=t.dtype, device="cuda")
        return big[1:-1, shift:shift + t.shape[1]].copy_(t)

    for pad in (0, 8, 13):
        _check({"y": gated_feed_forward(among(x, pad), among(wg, pad), among(wu, pad + 3), among(wd, pad))}, want)


# what is launched before the kernels has written the weights they read
@pytest.mark.gpu
def test_few_tokens_see_new_weights():
    x, wg, wu, wd, _ = _inputs(4, 2048, 5632, torch.bfloat16)
    want = gated_feed_forward(x, wg, wu, wd)
    new = [torch.empty_like(t) for t in (wg, wu, wd)]
    for _ in range(20):
        for t in new:
            t.zero_()
        for t, w in zip(new, (wg, wu, wd)):
            t.copy_(w)
        assert torch.equal(gated_feed_forward(x, *new), want)


# a device full of whole tiles and more, in bands of rows; long reductions that several pairs share
@pytest.mark.gpu
@pytest.mark.parametrize("tokens,width,hidden", [(5000, 520, 1100), (20000, 256, 136)])
def test_many_tiles(tokens, width, hidden):
    *args, dy = _inputs(tokens, width, hidden, torch.bfloat16, seed=1)
    want = _want(*args, dy, "silu", False, Rounding(torch.bfloat16))
    _check(_pass([t.requires_grad_() for t in args], dy), want)


@pytest.mark.gpu
@pytest.mark.parametrize("eight", [None, "int8"])
def test_what_is_kept_beyond_31_bits(eight):
    tokens, width, hidden = 400_000 if eight is None else 1_100_000, 16, 1000
    *args, dy = _inputs(tokens, width, hidden, torch.bfloat16)
    last = [args[0][-300:].clone(), *args[1:]]
    want = _want(*last, dy[-300:], "silu", eight is not None, Rounding(torch.bfloat16))
    x = args[0].requires_grad_()
    y = gated_feed_forward(x, *args[1:], checkpoint=eight)
    (dx,) = torch.autograd.grad(y, x, dy)
    _check({"y": y[-300:], "dx": dx[-300:]}, {k: want[k] for k in ("y", "dx")})


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradients_asked_for_alone(dtype):
    *args, dy = _inputs(150, 72, 200, dtype)
    every = _pass([t.clone().requires_grad_() for t in args], dy)
    for i, key in enumerate(("dx", "dw_gate", "dw_up", "dw_down")):
        some = [t.clone().requires_grad_(i == j) for j, t in enumerate(args)]
        (g,) = torch.autograd.grad(gated_feed_forward(*some), some[i], dy)
        assert torch.equal(g, every[key]), key


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradient_against_differences(dtype):
    *args, dy = _inputs(9, 24, 40, dtype, seed=5)
    at = [t.double() for t in args]
    bounds = _want(*args, dy, "gelu_tanh", False, Rounding(dtype))
    got = _pass([t.requires_grad_() for t in args], dy, activation="gelu_tanh")

    def loss(x, wg, wu, wd):
        return (((_act("gelu_tanh", x @ wg.T)[0] * (x @ wu.T)) @ wd.T) * dy.double()).sum()

    for i, key in enumerate(("dx", "dw_gate", "dw_up", "dw_down")):
        v = torch.randn(at[i].shape, dtype=torch.double, device="cuda", generator=torch.Generator(device="cuda").manual_seed(i))
        up, down = list(at), list(at)
        up[i], down[i] = at[i] + 1e-5 * v, at[i] - 1e-5 * v
        slope = (loss(*up) - loss(*down)) / 2e-5
        # 1e-5 squared times third derivatives of order 1 to 10 over a thousand numbers, and 2^-53 of the loss over 1e-5
        assert abs((got[key].double() * v).sum() - slope) <= (bounds[key][1] * v.abs()).sum() + 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_layouts(dtype):
    x, wg, wu, wd, dy = _inputs(90, 104, 136, dtype)
    want = _pass([t.clone().requires_grad_() for t in (x, wg, wu, wd)], dy)

    def wide(t, start):
        big = torch.zeros(t.shape[0], t.shape[1] + 24, dtype=dtype, device="cuda")[:, start:start + t.shape[1]]
        return big.copy_(t)

    for change in (lambda t: wide(t, 8), lambda t: wide(t, 3), lambda t: t.t().contiguous().t(), lambda t: torch.stack((t, t), -1)[..., 1]):
        some = [change(t).detach().requires_grad_() for t in (x, wg, wu, wd)]
        got = _pass(some, change(dy))
        for key in want:
            # fp32 products of another layout may be the library's
            assert torch.equal(got[key], want[key]) if dtype != torch.float32 else torch.allclose(got[key], want[key], rtol=1e-5, atol=1e-5), key
    some = [t.clone().requires_grad_() for t in (x.view(9, 2, 5, 104), wg, wu, wd)]
    y = gated_feed_forward(*some)
    assert y.shape == (9, 2, 5, 104) and torch.equal(y.view(90, 104), want["y"])
    y.backward(dy.view(9, 2, 5, 104))
    assert torch.equal(some[0].grad.view(90, 104), want["dx"]) and torch.equal(some[3].grad, want["dw_down"])
    line = gated_feed_forward(x[0], wg, wu, wd)
    assert line.shape == (104,)
    one = torch.ones((), dtype=dtype, device="cuda").expand(90, 104)
    a = [t.clone().requires_grad_() for t in (x, wg, wu, wd)]
    b = torch.autograd.grad(gated_feed_forward(*a), a, one)
    c = torch.autograd.grad(gated_feed_forward(*a), a, one.contiguous())
    assert all(torch.equal(p, q) for p, q in zip(b, c))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_infinities_nan_and_no_rows(dtype):
    x, wg, wu, wd, dy = _inputs(70, 64, 96, dtype)
    clean = gated_feed_forward(x, wg, wu, wd)
    y = x.clone()
    y[3, 5] = float("nan")
    y[66, 1] = float("inf")
    got = gated_feed_forward(y, wg, wu, wd)
    bad = torch.zeros(70, dtype=torch.bool, device="cuda")
    bad[3] = bad[66] = True
    assert not torch.isfinite(got[bad]).any() and torch.equal(got[~bad], clean[~bad])
    for eight in (None, "int8"):
        some = [t.clone().requires_grad_() for t in (y, wg, wu, wd)]
        grads = _pass(some, dy, checkpoint=eight)
        assert torch.isnan(grads["dx"][3]).all() and torch.isfinite(grads["dx"][~bad]).all() and torch.isnan(grads["dw_up"]).any()
        none = [x[:0].clone().requires_grad_(), *(w.clone().requires_grad_() for w in (wg, wu, wd))]
        empty = _pass(none, dy[:0], checkpoint=eight)
        assert empty["y"].shape == (0, 64) and empty["dx"].shape == (0, 64) and not empty["dw_gate"].any() and not empty["dw_down"].any()
    flat = torch.zeros_like(x).requires_grad_()
    for name in ("silu", "gelu_tanh"):
        assert not _pass([flat, *(w.clone().requires_grad_() for w in (wg, wu, wd))], dy, activation=name)["dw_down"].any()


@pytest.mark.gpu
@pytest.mark.parametrize("activation", ["silu", "gelu_tanh"])
def test_large_gates(activation):
    # far out both curves are the identity or zero, and so are their slopes one or zero
    x = torch.tensor([[-3e4, 1.0], [3e4, 1.0], [-80.0, 1.0], [80.0, 1.0]], device="cuda").bfloat16()
    eye = torch.eye(2, device="cuda").bfloat16()
    up = torch.tensor([[0.0, 1.0], [0.0, 1.0]], device="cuda").bfloat16()
    args = [t.clone().requires_grad_() for t in (x, eye, up, eye)]
    got = _pass(args, torch.ones_like(x), activation=activation)
    assert torch.equal(got["y"][:, 0].float().clamp(min=0), x[:, 0].float().clamp(min=0)) and (got["y"][:, 0].float() > -1e-30).all()
    one = _act(activation, torch.ones((), dtype=torch.double))[1]
    assert ((got["dx"][:, 0].float() - (x[:, 0] > 0).float()).abs() < 1e-30).all()
    assert all(torch.isfinite(t.float()).all() for t in got.values()) and one > 0


@pytest.mark.gpu
def test_what_is_kept():
    x, wg, wu, wd, _ = _inputs(512, 256, 704, torch.bfloat16)
    args = [t.requires_grad_() for t in (x, wg, wu, wd)]
    kept = {}
    for eight in (None, "int8"):
        seen = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append(t) or t, lambda t: t):
            gated_feed_forward(*args, checkpoint=eight)
        kept[eight] = sum(t.numel() * t.element_size() for t in seen if not any(t is w or t.shape == w.shape for w in (wg, wu, wd)))
    assert kept[None] == 512 * (256 * 2 + 704 * 6)
    assert kept["int8"] == 512 * (256 + 256 // 16 + 2 * (704 + 704 // 16))


@pytest.mark.gpu
def test_streams_graphs_autocast_and_double_backward():
    *args, dy = _inputs(300, 256, 704, torch.bfloat16)
    want = gated_feed_forward(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = gated_feed_forward(*args)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = gated_feed_forward(*args)
    args[0].mul_(0.5)
    graph.replay()
    assert torch.equal(again, gated_feed_forward(*args)) and not torch.equal(again, want)
    block = GatedFeedForward(256, 704, device="cuda")
    x = torch.randn(4, 75, 256, device="cuda", requires_grad=True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = block(x)
    assert y.dtype == torch.bfloat16 and y.shape == x.shape
    y.float().square().mean().backward()
    assert block.w_gate.grad.dtype == torch.float32 and torch.isfinite(block.w_gate.grad).all() and x.grad.dtype == torch.float32
    a = [t.clone().requires_grad_() for t in args]
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(gated_feed_forward(*a).float().sum(), a, create_graph=True)


@pytest.mark.gpu
def test_repeated_calls_are_bit_equal():
    *args, dy = _inputs(2000, 512, 1408, torch.bfloat16)
    args = [t.requires_grad_() for t in args]
    first = _pass(args, dy, checkpoint="int8")
    for _ in range(5):
        again = _pass(args, dy, checkpoint="int8")
        assert all(torch.equal(first[k], again[k]) for k in first)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,width,hidden", [(333, 1000, 2731), (40, 520, 4001), (2000, 64, 130), (100, 999, 515)])
def test_copied_rows_of_calls_one_after_another(tokens, width, hidden):
    # what is copied for one call lies where an earlier one's copies, parts and h lay, which its kernels may still read
    sets = [_inputs(tokens, width, hidden, torch.bfloat16, seed=i)[:4] for i in range(3)]
    want = []
    for args in sets:
        want.append(gated_feed_forward(*args))
        torch.cuda.synchronize()
    got = [gated_feed_forward(*sets[i % 3]) for i in range(60)]
    assert all(torch.equal(g, want[i % 3]) for i, g in enumerate(got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [gated_feed_forward(*args) for args in sets]
    for _ in range(5):
        graph.replay()
    assert all(torch.equal(g, w) for g, w in zip(got, want))


@pytest.mark.gpu
def test_memory_of_copies_beside_a_product_is_taken_before_it():
    # these copies wait for nothing that runs, so a block that is freed after the product before them was launched may not be theirs
    tokens, width, hidden = 333, 1024, 2731
    x, wg, wu, wd = _inputs(tokens, width, hidden, torch.bfloat16)[:4]
    gated_feed_forward(x, wg, wu, wd)
    torch.cuda.synchronize()
    torch.cuda.memory._record_memory_history(max_entries=1000)
    try:
        gated_feed_forward(x, wg, wu, wd)
        trace = torch.cuda.memory._snapshot()["device_traces"][0]
    finally:
        torch.cuda.memory._record_memory_history(enabled=None)
    sizes = [e["size"] for e in trace if e["action"] == "alloc"]
    copies, h = width * 2736 * 2, tokens * 2752 * 2
    assert sizes.count(copies) == 1 and sizes.count(h) == 1 and sizes.index(copies) < sizes.index(h)


@pytest.mark.gpu
def test_threads_that_share_a_stream():
    from mccl_b200.ops.linear import linear
    x, wg, wu, wd = _inputs(333, 1024, 2731, torch.bfloat16)[:4]    # w_down is copied beside the first product
    y, vg, vu, vd = _inputs(1000, 640, 2112, torch.bfloat16, seed=1)[:4]  # reductions that pairs share: a launch that adds them up
    a, b, _, _, _ = _inputs(64, 1024, 4096, torch.float32, seed=2)
    calls = [lambda: gated_feed_forward(x, wg, wu, wd), lambda: gated_feed_forward(y, vg, vu, vd), lambda: linear(a, b)]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    stream, wrong, ready = torch.cuda.current_stream(), [], threading.Barrier(len(calls))

    def work(i):
        try:
            with torch.no_grad(), torch.cuda.stream(stream):
                ready.wait()
                for _ in range(40):
                    got = [calls[i]() for _ in range(10)]
                    if not all(torch.equal(g, want[i]) for g in got):
                        wrong.append(i)
        except Exception as e:  # noqa: BLE001
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.gpu
def test_waits_that_run_out_are_reported_and_leave_nan():
    # in a process of its own: the report is one for the whole device
    code = """
import torch, mccl_b200
from mccl_b200.ops.gated import gated_feed_forward
native = mccl_b200.require_native()
x, w, d = (torch.randn(*s, device="cuda").bfloat16() for s in ((300, 256), (512, 256), (256, 512)))
y = native._gated_with_limit(x, w, w, d, 0)
torch.cuda.synchronize()
assert torch.isnan(y).all()
try:
    gated_feed_forward(x, w, w, d)
except RuntimeError as e:
    assert "ran out" in str(e)
else:
    raise AssertionError("not reported")
y = gated_feed_forward(x, w, w, d)
assert torch.isfinite(y).all()
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.gpu
def test_refusals():
    x, wg, wu, wd, _ = _inputs(4, 16, 24, torch.bfloat16)
    for args in ((x.float(), wg, wu, wd), (x.double(), wg.double(), wu.double(), wd.double()), (x, wg[:, :8], wu, wd), (x, wg[:8], wu, wd), (x, wg, wu, wd.t()),
                 (x, wg, wu, wd.cpu()), (x, wg[0], wu, wd), (x[:, :0], wg[:, :0], wu[:, :0], wd[:0]), (x.sum(), wg, wu, wd)):
        with pytest.raises(RuntimeError, match="MCCL"):
            gated_feed_forward(*args)
    with pytest.raises(RuntimeError, match="transforms"):
        torch.func.vmap(lambda a: gated_feed_forward(a, wg, wu, wd))(x[None])


def test_refusals_of_options():
    t = torch.zeros(2, 2)
    for kw in (dict(activation="relu"), dict(checkpoint="int4"), dict(checkpoint=True)):
        with pytest.raises(ValueError):
            gated_feed_forward(t, t, t, t, **kw)
        with pytest.raises(ValueError):
            GatedFeedForward(2, 2, **kw)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("activation", ["silu", "gelu_tanh"])
def test_cpu_form(activation, eight):
    *args, dy = _inputs(13, 70, 130, torch.float32, device="cpu")
    want = _want(*args, dy, activation, eight, Rounding(torch.float32))
    _check(_pass([t.requires_grad_() for t in args], dy, activation=activation, checkpoint="int8" if eight else None), want)
    block = GatedFeedForward(70, 130, activation=activation, checkpoint="int8" if eight else None)
    x = torch.randn(2, 3, 70, requires_grad=True)
    block(x).sum().backward()
    assert x.grad.shape == x.shape and block.w_down.grad.shape == (70, 130) and "hidden=130" in repr(block)
    assert mccl_b200.__version__


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_autocast_is_a_call_with_tensors_of_its_type(checkpoint, device):
    *args, dy = _inputs(13, 72, 130, torch.float32, device=device)
    low = [t.bfloat16().requires_grad_() for t in args]
    y = gated_feed_forward(*low, checkpoint=checkpoint)
    want = torch.autograd.grad(y, low, dy.bfloat16())
    args = [t.requires_grad_() for t in args]
    with torch.autocast(device, dtype=torch.bfloat16):
        z = gated_feed_forward(*args, checkpoint=checkpoint)
    got = torch.autograd.grad(z, args, dy.bfloat16())
    assert torch.equal(y, z) and all(g.dtype == torch.float32 and torch.equal(g, w.float()) for g, w in zip(got, want))


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("checkpoint", [None, "int8"])
@pytest.mark.parametrize("tokens,width,hidden", [(5, 8, 24), (256, 512, 704)])
def test_backward_inside_of_an_autocast_region(tokens, width, hidden, checkpoint, dtype, device):
    *args, dy = _inputs(tokens, width, hidden, dtype, device=device)
    args = [t.requires_grad_() for t in args]
    y = gated_feed_forward(*args, checkpoint=checkpoint)
    want = torch.autograd.grad(y, args, dy, retain_graph=True)
    with torch.autocast(device, dtype=torch.bfloat16):
        got = torch.autograd.grad(y, args, dy)
        assert torch.is_autocast_enabled(device)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_the_cpu_form_refuses_what_the_kernels_refuse():
    x, wg, wu, wd, _ = _inputs(4, 16, 24, torch.float32, device="cpu")
    gated_feed_forward(x[0], wg, wu, wd), gated_feed_forward(x.double(), wg.double(), wu.double(), wd.double())
    for args in ((x.half(), wg, wu, wd), (x, wg[:, :8], wu, wd), (x, wg[:8], wu, wd), (x, wg, wu[:1], wd), (x, wg[:1], wu, wd), (x, wg, wu, wd[:5]), (x, wg, wu, wd.t()),
                 (x, wg[0], wu, wd), (x[:, :0], wg[:, :0], wu[:, :0], wd[:0]), (x, wg[:0], wu[:0], wd[:, :0]), (x.sum(), wg, wu, wd)):
        with pytest.raises(ValueError, match="gated_feed_forward"):
            gated_feed_forward(*args)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 4, 8, 40])
def test_float32_gates_far_out(tokens):
    # h = silu(z), of its own kernels for few tokens and between two products.  The exponential is within 2 units in the last place, 4
    # times 2^-24; its sum with one, the quotient and the product with z round once each; the other products are with ones and zeros.
    z = torch.linspace(-85, 85, 960, device="cuda")
    eye, up = torch.eye(2, device="cuda"), torch.tensor([[0.0, 1.0], [0.0, 1.0]], device="cuda")
    x = torch.stack((z, torch.ones_like(z)), 1)
    got = torch.cat([gated_feed_forward(x[i:i + tokens], eye, up, eye) for i in range(0, 960, tokens)])[:, 0].double()
    want = z.double() * torch.sigmoid(z.double())
    assert ((got - want).abs() <= want.abs() * 8 * 2.0 ** -24).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("activation", ["silu", "gelu_tanh"])
def test_gradients_at_a_gate_of_one(activation, dtype):
    # z = 1: the gradient of x's first number is act'(1), of its second act(1)
    x = torch.tensor([[1.0, 1.0]], dtype=dtype, device="cuda")
    gate, up = torch.tensor([[1.0, 0.0]], dtype=dtype, device="cuda"), torch.tensor([[0.0, 1.0]], dtype=dtype, device="cuda")
    down = torch.ones(2, 1, dtype=dtype, device="cuda")
    args = [t.requires_grad_() for t in (x, gate, up, down)]
    got = _pass(args, torch.tensor([[1.0, 0.0]], dtype=dtype, device="cuda"), activation=activation)
    a, slope = (v.item() for v in _act(activation, torch.ones((), dtype=torch.double)))
    # two roundings of the type at most (an operand's and the result's), the gate's 2^-16 (fp32 2^-20)
    near = 2.5 * ROUNDOFF[dtype] + (2.0 ** -16 if dtype != torch.float32 else 2.0 ** -20)
    for value, want in ((got["y"][0, 0], a), (got["y"][0, 1], a), (got["dx"][0, 0], slope), (got["dx"][0, 1], a), (got["dw_gate"][0, 0], slope),
                        (got["dw_gate"][0, 1], slope), (got["dw_up"][0, 0], a), (got["dw_down"][0, 0], a)):
        assert abs(value.item() - want) <= near * want
    assert got["dw_down"][1, 0].item() == 0


@pytest.mark.gpu
def test_float32_products_are_torchs_where_tf32_is_allowed():
    native = mccl_b200.require_native()
    *args, dy = _inputs(256, 1024, 2816, torch.float32)
    args = [t.requires_grad_() for t in args]
    was = torch.backends.cuda.matmul.allow_tf32
    counts = []
    try:
        for allowed in (False, True):
            torch.backends.cuda.matmul.allow_tf32 = allowed
            y = gated_feed_forward(*args)
            before = native._kernel_launches()
            torch.autograd.grad(y, args, dy)
            counts.append(native._kernel_launches() - before)
    finally:
        torch.backends.cuda.matmul.allow_tf32 = was
    # what stands between the products is two launches; each product has others of its own
    assert counts[0] > 2 and counts[1] == 2
