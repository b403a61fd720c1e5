"""Activation checkpoints in 8 bits against their formula."""
import pytest
import torch

import mccl_b200
from mccl_b200.ops import checkpoint
from mccl_b200.ops.checkpoint import GROUP, Packed8, pack8, unpack8

TYPES = [torch.float32, torch.float16, torch.bfloat16]
ROUNDOFF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _formula(x):
    """Codes and scales in 32 bits, row by row and group by group."""
    rows = x.detach().float().cpu().reshape(-1, x.shape[-1])
    codes = torch.zeros(rows.shape, dtype=torch.int8)
    scales = torch.zeros(rows.shape[0], -(-rows.shape[1] // GROUP))
    for g in range(scales.shape[1]):
        v = rows[:, g * GROUP:(g + 1) * GROUP]
        most = v.abs().amax(1)
        ok = torch.isfinite(most) & (most >= 2.0 ** -100)
        top = torch.full_like(most, 127.0)
        codes[:, g * GROUP:(g + 1) * GROUP] = torch.where(ok[:, None], torch.round(v * (top / most)[:, None]), 0.0).to(torch.int8)
        scales[:, g] = torch.where(ok, most / top, torch.where(most < 2.0 ** -100, 0.0, float("nan")))
    return codes, scales


def _data(shape, dtype, device, seed=0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=gen) * torch.exp(2 * torch.randn(shape[-1:], generator=gen))
    return x.to(dtype).to(device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 63), (3, 64), (5, 65), (2, 7, 130), (257, 1000), (33, 4096), (1000, 17), (4, 0), (0, 5), (9,)])
def test_codes_scales_and_values_are_the_formulas(shape, dtype, device):
    x = _data(shape, dtype, device)
    p = pack8(x)
    back = unpack8(p)
    assert back.shape == x.shape and back.dtype == dtype and back.is_contiguous()
    if x.numel() == 0:
        return
    codes, scales = _formula(x)
    cols = shape[-1]
    assert torch.equal(p.codes[:, :cols].cpu(), codes) and not p.codes[:, cols:].any()
    assert torch.equal(p.scales.cpu(), scales)
    each = scales.repeat_interleave(GROUP, 1)[:, :cols]
    assert torch.equal(back.cpu().reshape(-1, cols), (codes.float() * each).to(dtype))
    # half a step (a code's product and the scale round by 2^-24 each, up to 127 steps from zero), and the type's own rounding
    off = (back.double().cpu().reshape(-1, cols) - x.double().cpu().reshape(-1, cols)).abs()
    assert (off <= each.double() * (0.5 + 128 * 2.0 ** -23) + each.double() * 127 * ROUNDOFF[dtype] + 2.0 ** -25).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
def test_infinities_nan_zeros_and_the_smallest(dtype, device):
    x = torch.ones(6, 3 * GROUP, dtype=dtype, device=device)
    x[0, 5] = float("inf")
    x[1, GROUP + 63] = float("-inf")
    x[2, 2 * GROUP] = float("nan")
    x[3] = 0
    x[4] = torch.finfo(dtype).max
    x[5] = torch.finfo(dtype).smallest_normal
    back = unpack8(pack8(x)).float()
    bad = torch.zeros(6, 3, dtype=torch.bool, device=device)
    bad[0, 0] = bad[1, 1] = bad[2, 2] = True
    assert torch.equal(torch.isnan(back).view(6, 3, GROUP), bad[..., None].expand(6, 3, GROUP))
    assert (back[:3][~torch.isnan(back[:3])] - 1).abs().max() <= 127 * 2.0 ** -23
    assert not back[3].any()
    # the largest number of a type may come back 2^-23 above itself; in the 16-bit types and in 32 bits that rounds to itself or to
    # the next number, infinity
    assert (back[4] >= torch.finfo(dtype).max * (1 - 2.0 ** -22)).all()
    assert (back[5] == 0).all() if torch.finfo(dtype).smallest_normal < 2.0 ** -100 else (back[5] > 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_views(dtype):
    base = _data((70, 401), dtype, "cuda")
    for x in (base[:, 1:400], base[:, 8:136], base[::2, 16:], base.t(), base[:1].expand(9, 401), base[:, :1], base[3:4, 5:], base[:, ::2]):
        codes, scales = _formula(x)
        p = pack8(x)
        assert torch.equal(p.codes[:, :x.shape[1]].cpu(), codes) and torch.equal(p.scales.cpu(), scales)
        assert torch.equal(unpack8(p), unpack8(pack8(x.contiguous())))


@pytest.mark.gpu
def test_another_stream_and_a_graph():
    x = _data((300, 700), torch.bfloat16, "cuda")
    want = unpack8(pack8(x))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = unpack8(pack8(x))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = unpack8(pack8(x))
    x.neg_()
    graph.replay()
    assert torch.equal(again, -want)


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [65536, 65541])
def test_more_than_two_to_the_31_numbers(cols):
    rows = 33000
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    x[-3:] = _data((3, cols), torch.bfloat16, "cuda", seed=4)
    x[5] = 1
    back = unpack8(pack8(x))
    assert torch.equal(back[-3:], unpack8(pack8(x[-3:].clone()))) and not back[-4].any() and not back[6].any()
    assert ((back[5] - 1).abs() <= 2.0 ** -8).all()


def test_refusals_on_cpu():
    with pytest.raises(TypeError, match="float32, float16 or bfloat16"):
        pack8(torch.zeros(3, dtype=torch.float64))
    with pytest.raises(TypeError):
        pack8(torch.zeros(3, dtype=torch.int32))


@pytest.mark.gpu
def test_refusals():
    native = mccl_b200.require_native()
    with pytest.raises(TypeError):
        pack8(torch.zeros(3, device="cuda", dtype=torch.float64))
    p = pack8(torch.zeros(4, 100, device="cuda"))
    for broken in (p._replace(shape=(5, 100)), p._replace(shape=(4, 99 + 30)), p._replace(scales=p.scales[:3]), p._replace(codes=p.codes[:, :96]),
                   p._replace(codes=p.codes.to(torch.uint8)), p._replace(scales=p.scales.double()), p._replace(shape=(4, -100)),
                   p._replace(dtype=torch.float64), p._replace(scales=p.scales.cpu())):
        with pytest.raises(RuntimeError, match="MCCL"):
            unpack8(broken)
    with pytest.raises(RuntimeError, match="MCCL"):
        native._pack8(torch.zeros(3))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bias", [False, True])
def test_linear_keeps_its_input_in_8_bits(bias, device):
    torch.manual_seed(1)
    x, w = torch.randn(3, 37, 130, device=device, requires_grad=True), torch.randn(50, 130, device=device, requires_grad=True)
    b = torch.randn(50, device=device, requires_grad=True) if bias else None
    g = torch.randn(3, 37, 50, device=device)
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        y = checkpoint.linear(x, w, b)
    assert sum(t.numel() * t.element_size() for t in kept if t.shape != w.shape) <= 1.3 * x.numel()
    y.backward(g)
    x64, w64, g64 = x.detach().double(), w.detach().double(), g.double()
    seen = unpack8(pack8(x)).double()
    want = x64 @ w64.T + (b.detach().double() if bias else 0)

    # fp32 products (sums of 130, 50 and 111 terms): each term and each sum rounds by 2^-24 of the terms' absolute sum at most
    def near(a, r, size, depth):
        return ((a.detach().double() - r).abs() <= size * (depth + 2) * 2.0 ** -24).all()

    assert near(y, want, x64.abs() @ w64.abs().T + (b.detach().abs().double() if bias else 0), 131)
    assert near(x.grad, g64 @ w64, g64.abs() @ w64.abs(), 50)
    rows, again = g64.flatten(0, 1), seen.flatten(0, 1)
    assert near(w.grad, rows.T @ again, rows.abs().T @ again.abs(), 111)
    if bias:
        assert near(b.grad, rows.sum(0), rows.abs().sum(0), 111)
    with pytest.raises(RuntimeError):
        y = checkpoint.linear(x, w, b)
        torch.autograd.grad(torch.autograd.grad(y.sum(), w, create_graph=True)[0].sum(), x)


@pytest.mark.gpu
def test_linear_under_autocast():
    torch.manual_seed(2)
    x, w = torch.randn(64, 128, device="cuda", requires_grad=True), torch.randn(96, 128, device="cuda", requires_grad=True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = checkpoint.linear(x, w)
    assert y.dtype == torch.bfloat16
    y.float().sum().backward()
    assert x.grad.dtype == torch.float32 and w.grad.dtype == torch.float32 and torch.isfinite(w.grad).all()
    seen = unpack8(pack8(x.detach().bfloat16())).double()
    want = torch.ones(64, 96, device="cuda", dtype=torch.double).T @ seen
    # a bf16 product of 64 terms that are added up in fp32 and rounded once
    assert ((w.grad.double() - want).abs() <= want.abs() * 2.0 ** -8 + seen.abs().sum(0) * 66 * 2.0 ** -23).all()


@pytest.mark.parametrize("device", DEVICES)
def test_autocast_leaves_float64(device):
    from mccl_b200.ops.gated import gated_feed_forward
    x, w = _data((4, 8), torch.float32, device).double(), _data((6, 8), torch.float32, device, seed=1).double()
    want = x @ w.t()
    with torch.autocast(device, dtype=torch.bfloat16):
        with torch.no_grad():
            assert torch.nn.functional.linear(x, w).dtype == torch.float64
            assert torch.allclose(checkpoint.linear(x, w), want, rtol=1e-12, atol=1e-12)
            if device == "cpu":
                assert gated_feed_forward(x, w, w, w.t()).dtype == torch.float64
            else:
                with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
                    gated_feed_forward(x, w, w, w.t())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
def test_backward_inside_of_an_autocast_region(dtype, device):
    x, w = _data((37, 130), dtype, device).requires_grad_(), _data((50, 130), dtype, device, seed=1).requires_grad_()
    y = checkpoint.linear(x, w)
    dy = _data((37, 50), dtype, device, seed=2)
    want = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
    with torch.autocast(device, dtype=torch.bfloat16):
        got = torch.autograd.grad(y, (x, w), dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_the_cpu_form_refuses_what_the_kernels_refuse():
    p = pack8(torch.ones(4, 100))
    for broken in (p._replace(shape=(5, 100)), p._replace(shape=(4, 99 + 30)), p._replace(shape=(8, 50)), p._replace(scales=p.scales[:3]),
                   p._replace(scales=p.scales[:1]), p._replace(codes=p.codes[:, :96]), p._replace(codes=p.codes[:1]), p._replace(codes=p.codes.to(torch.uint8)),
                   p._replace(scales=p.scales.double()), p._replace(shape=(4, -100)), p._replace(dtype=torch.float64)):
        with pytest.raises(ValueError, match="unpack8"):
            unpack8(broken)


@pytest.mark.parametrize("device", DEVICES)
def test_nothing_is_packed_where_no_gradient_can_follow(device, monkeypatch):
    from mccl_b200.models import gated_tiny
    from mccl_b200.ops import gated
    packed = []

    def counted(x):
        packed.append(x.shape)
        return pack8(x)

    monkeypatch.setattr(checkpoint, "pack8", counted)
    monkeypatch.setattr(gated, "pack8", counted)
    model = gated_tiny(checkpoint="int8").to(device)
    ids = torch.randint(0, 1024, (2, 5), device=device)
    model.generate(ids, 2)
    with torch.no_grad(), torch.autocast(device, dtype=torch.bfloat16):
        model(ids)
    model.requires_grad_(False)
    model(ids)
    x, w = _data((7, 64), torch.float32, device), _data((5, 64), torch.float32, device, seed=1)
    with torch.inference_mode():
        want = checkpoint.linear(x, w.requires_grad_())
    assert not packed
    assert torch.equal(checkpoint.linear(x, w), want) and packed == [(7, 64)]
    # of types that the codes don't have, too
    with torch.no_grad():
        assert checkpoint.linear(x.double(), w.double()).dtype == torch.float64
