"""Layer norm with the sum before it: results and gradients against 64 bits, layouts, modes, refusals."""
import math

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from mccl_b200.ops.layer_norm import LayerNorm, layer_norm

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
EPS = 1e-5


def _inputs(rows, cols, dtype, stream, out, affine, device, seed=0, mean=0.3):
    gen = torch.Generator().manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    t = {"x": (randn(rows, cols) + mean).to(dtype)}
    if stream is not None:
        t["residual"] = (2 * randn(rows, cols) + mean).to(stream)
        t["ds"] = randn(rows, cols).to(stream)
    if affine is not None:
        t["weight"], t["bias"] = (1 + 0.3 * randn(cols)).to(affine), (0.2 * randn(cols)).to(affine)
    t["dy"] = randn(rows, cols).to(out)
    return {k: v.to(device) for k, v in t.items()}


def _call(t, out, grad=True):
    leaves = [t[k].requires_grad_() for k in ("x", "weight", "bias", "residual") if k in t] if grad else []
    result = layer_norm(t["x"], t.get("weight"), t.get("bias"), eps=EPS, residual=t.get("residual"), dtype=out)
    result = result if "residual" in t else (result,)
    if not grad:
        return list(result), []
    return [r.detach() for r in result], list(torch.autograd.grad(result, leaves, [t["dy"], t["ds"]] if "residual" in t else [t["dy"]]))


def _check(t, out, results, grads):
    """Every result within what its roundings allow.

    The mean and the mean square are sums of n numbers, 32 at most a thread and the rest in trees: 64 roundings of a mean of magnitudes are
    above both, so u = (s - mean) rstd is off by E = 64 U (mean|s| rstd + |u|) at most.  Sums of products of u inherit that; their
    own roundings are below 128 U of the sum of magnitudes, the weights' below 256 U (3000 rows: 7 a thread, 8 teams, 56 parts, 8 warps).
    """
    t = {k: v.detach().cpu() for k, v in t.items()}
    s = t["x"].double()
    if "residual" in t:
        kept = (t["x"].float() + t["residual"].float()).to(t["residual"].dtype)
        assert torch.equal(results[1].cpu(), kept)
        s = kept.double()
    w, b = (t[k].double() if k in t else torch.tensor(v).double() for k, v in (("weight", 1.0), ("bias", 0.0)))
    size = s.abs().mean(-1, keepdim=True)
    mean = s.mean(-1, keepdim=True)
    rstd = (((s - mean) ** 2).mean(-1, keepdim=True) + EPS).rsqrt()
    u = (s - mean) * rstd
    E = 64 * U * (size * rstd + u.abs())
    y = u * w + b

    def near(got, want, bound, what):
        assert got.shape == want.shape, what
        bound = bound + HALF[got.dtype] * (want.abs() + bound)
        if got.dtype is torch.float16:
            bound = bound + 2.0 ** -25  # half of the smallest subnormal
        worst = ((got.double().cpu() - want).abs() - bound).max() if got.numel() else torch.tensor(0.0)
        assert worst <= 0, (what, float(worst))

    assert results[0].dtype is (out or t["x"].dtype)
    near(results[0], y, E * w.abs() + 3 * U * ((u * w).abs() + b.abs()), "y")
    if not grads:
        return
    dy = t["dy"].double()
    g = dy * w
    first, second = g.mean(-1, keepdim=True), (g * u).mean(-1, keepdim=True)
    sizes = g.abs() + g.abs().mean(-1, keepdim=True) + u.abs() * (g * u).abs().mean(-1, keepdim=True)
    dx = rstd * (g - first - u * second)
    bound = rstd * (128 * U * sizes + E * (g * u).abs().mean(-1, keepdim=True) + u.abs() * (g.abs() * E).mean(-1, keepdim=True))
    if "residual" in t:
        dx, bound = dx + t["ds"].double(), bound + 2 * U * t["ds"].double().abs()
    grads = list(grads)
    near(grads.pop(0), dx, bound, "dx")
    if "weight" in t:
        near(grads.pop(0), (dy * u).sum(0), (256 * U * (dy * u).abs() + dy.abs() * E).sum(0), "dweight")
        near(grads.pop(0), dy.sum(0), (256 * U * dy.abs()).sum(0), "dbias")
    if "residual" in t:
        near(grads.pop(0), dx, bound, "dresidual")


SIZES = [(1, 1), (3, 2), (2, 7), (5, 8), (37, 31), (64, 64), (9, 255), (7, 256), (3, 257), (130, 1000), (33, 1024), (21, 1723), (3000, 72), (5, 4096),
         (4, 4097), (3, 4104), (2, 8192), (3, 8193), (2, 8200), (2, 16384), (3, 16385), (2, 20008)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("dtype,stream,out,affine", [
    (torch.float32, None, None, torch.float32), (torch.bfloat16, torch.float32, torch.bfloat16, torch.float32), (torch.float16, torch.float16, None, torch.float16),
])
def test_results_and_gradients(device, rows, cols, dtype, stream, out, affine):
    t = _inputs(rows, cols, dtype, stream, out or dtype, affine, device)
    _check(t, out, *_call(t, out))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("stream", [None, "same", torch.float32])
@pytest.mark.parametrize("out", [None, torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("affine", [None, "same", torch.float32])
@pytest.mark.parametrize("cols", [40, 43])
def test_types(device, dtype, stream, out, affine, cols):
    stream, affine = (dtype if v == "same" else v for v in (stream, affine))
    t = _inputs(6, cols, dtype, stream, out or dtype, affine, device, seed=1)
    _check(t, out, *_call(t, out))
    _check(t, out, _call({k: v.detach() for k, v in t.items()}, out, grad=False)[0], [])


@pytest.mark.parametrize("device", DEVICES)
def test_a_large_mean_costs_nothing(device):
    t = _inputs(8, 1000, torch.float32, None, torch.float32, torch.float32, device, mean=1000.0)
    results, grads = _call(t, None)
    _check(t, None, results, grads)


@pytest.mark.parametrize("device", DEVICES)
def test_rows_alike_rows_not_finite_and_no_rows(device):
    x = torch.ones(4, 24, device=device)
    x[1], x[2, 3] = math.nan, math.inf
    x[3] = torch.arange(24.0)
    w, b = torch.full((24,), 2.0, device=device), torch.full((24,), 0.5, device=device)
    y = layer_norm(x, w, b)
    assert torch.equal(y[0], b) and torch.isnan(y[1]).all() and torch.isnan(y[2]).all() and torch.isfinite(y[3]).all()
    w.requires_grad_(), b.requires_grad_()
    none = torch.zeros(0, 24, device=device, requires_grad=True)
    y, s = layer_norm(none, w, b, residual=torch.zeros(0, 24, device=device))
    grads = torch.autograd.grad((y.sum(), s.sum()), (none, w, b))
    assert y.shape == s.shape == (0, 24) and all(float(g.abs().sum()) == 0 for g in grads)
    assert layer_norm(torch.zeros(3, 0, 24, device=device)).shape == (3, 0, 24)


@pytest.mark.parametrize("device", DEVICES)
def test_one_of_the_gradients_alone(device):
    t = _inputs(9, 100, torch.bfloat16, torch.float32, torch.bfloat16, torch.float32, device)
    full = _call(t, None)[1]
    names = ["x", "weight", "bias", "residual"]
    for i, name in enumerate(names):
        for k in names:
            t[k] = t[k].detach().requires_grad_(k == name)
        out = layer_norm(t["x"], t["weight"], t["bias"], residual=t["residual"])
        (g,) = torch.autograd.grad(out, [t[name]], [t["dy"], t["ds"]])
        assert torch.equal(g, full[i]), name
    for which in (0, 1):  # only one of the results is used
        out = layer_norm(t["x"], t["weight"], t["bias"], residual=t["residual"])
        (g,) = torch.autograd.grad(out[which], [t["residual"]], [t[("dy", "ds")[which]]])
        if which:
            assert torch.equal(g, t["ds"])
        else:
            other = {k: v.detach() for k, v in t.items()}
            other["ds"] = torch.zeros_like(t["ds"])
            assert torch.equal(g, _call(other, None)[1][3])


@pytest.mark.parametrize("device", DEVICES)
def test_layouts(device):
    gen = torch.Generator().manual_seed(4)
    base = torch.randn(6, 5, 203, generator=gen).to(device)
    w = torch.randn(100, generator=gen).to(device)
    dy = torch.randn(6, 5, 100, generator=gen).to(device)

    def both(x, residual, dy):
        x, residual = x.detach().requires_grad_(), residual.detach().requires_grad_()
        out = layer_norm(x, w, residual=residual)
        return [o.detach() for o in out] + list(torch.autograd.grad(out, (x, residual), (dy, torch.ones_like(dy))))

    views = [base[:, :, :100], base[:, :, 3:103], base[:, :, 0:200:2], base.transpose(0, 1)[:, :, 1:101].transpose(0, 1), base[:, :1, 4:104].expand(6, 5, 100),
             base[0, 0, :100].expand(6, 5, 100)]
    for x in views:
        for residual in views:
            want = both(x.contiguous().clone(), residual.contiguous().clone(), dy.clone())
            got = both(x, residual, dy)
            # a run of another length changes the order of a row's sums, not what each may be off by
            assert all(torch.allclose(a, b, rtol=0, atol=300 * U * float(b.abs().max())) for a, b in zip(got, want))
    x = base[:, :, :100].detach().requires_grad_()
    g1 = torch.autograd.grad(layer_norm(x, w).sum(), x)[0]  # a gradient of stride zero
    g2 = torch.autograd.grad(layer_norm(x, w), x, torch.ones_like(dy))[0]
    assert torch.allclose(g1, g2, rtol=0, atol=300 * U * float(w.abs().max()) * float(base.abs().max()))
    assert layer_norm(base[0, 0, :100]).shape == (100,)


@pytest.mark.parametrize("device", DEVICES)
def test_gradients_are_those_of_differences(device):
    t = _inputs(5, 60, torch.float32, torch.float32, torch.float32, torch.float32, device, seed=6)
    _, grads = _call(t, None)
    gen = torch.Generator().manual_seed(9)
    for name, grad in zip(("x", "weight", "bias", "residual"), grads):
        way = torch.randn(t[name].shape, generator=gen).to(device)
        h = 2.0 ** -7

        def value(sign):
            moved = {k: v.detach() for k, v in t.items()}
            moved[name] = moved[name] + sign * h * way
            results, _ = _call(moved, None, grad=False)
            return sum(float((r.double() * d.double()).sum()) for r, d in zip(results, (t["dy"], t["ds"])))

        got, want = (value(1) - value(-1)) / (2 * h), float((grad.double() * way.double()).sum())
        # 300 results, each off by some 100 U of its size of a few, over h; the third derivative times h^2 / 6: sums of 300 terms of size one
        assert abs(got - want) <= 300 * 4 * 100 * U / h + 300 * 3 * h * h


@pytest.mark.parametrize("device", DEVICES)
def test_module_and_modes(device):
    gen = torch.Generator().manual_seed(3)
    x, other = (torch.randn(7, 48, generator=gen).to(device) for _ in range(2))
    m = LayerNorm(48).to(device)
    torch.nn.init.normal_(m.weight)
    ref = torch.nn.LayerNorm(48).to(device)
    ref.load_state_dict(m.state_dict())
    m.requires_grad_(False), ref.requires_grad_(False)
    assert torch.allclose(m(x), ref(x), rtol=0, atol=200 * U * float(ref(x).abs().max()))
    y, s = m(x, other, torch.bfloat16)
    assert y.dtype is torch.bfloat16 and torch.equal(s, x + other)
    assert LayerNorm(48, elementwise_affine=False)(x.cpu()).shape == x.shape and LayerNorm(48, bias=False).bias is None
    with torch.autocast(device, dtype=torch.bfloat16):
        assert m(x).dtype is torch.float32 and torch.equal(m(x), m(x))
    for pre in (False, True):
        traced = make_fx(lambda t: layer_norm(t, m.weight.detach(), m.bias.detach()), pre_dispatch=pre)(x)
        assert torch.allclose(traced(other), ref(other), rtol=0, atol=200 * U * float(ref(other).abs().max()))
    with pytest.raises(ValueError):
        LayerNorm((3, 48))


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    x = torch.randn(4, 16, device=device)
    w = torch.ones(16, device=device)
    kind = ValueError if device == "cpu" else RuntimeError
    for args, kw in [((x.double(),), {}), ((x.long(),), {}), ((x[0, 0],), {}), ((x[:, :0],), {}), ((x, w[:8]), {}), ((x, w.half()), {}), ((x, w.bfloat16(), w), {}),
                     ((x.half(), w.half(), w), {}), ((x, torch.ones(32, device=device)[::2]), {}), ((x, w[None]), {}), ((x,), dict(residual=x[:2])), ((x,), dict(residual=x.half())),
                     ((x.half(),), dict(residual=x.bfloat16())), ((x,), dict(dtype=torch.float64)), ((x,), dict(dtype=torch.int8)), ((x,), dict(eps=0.0)),
                     ((x,), dict(eps=math.inf)), ((x,), dict(eps=math.nan))]:
        with pytest.raises(kind, match="layer_norm"):
            layer_norm(*args, **kw)


@pytest.mark.gpu
def test_refusals_of_the_kernels(cuda_device):
    x = torch.randn(4, 16, device=cuda_device, requires_grad=True)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        layer_norm(x, torch.ones(16))
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(layer_norm(x).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="layer_norm"):
        torch.func.vmap(lambda t: layer_norm(t))(x.detach())
    y = layer_norm(x)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(lambda t: torch.autograd.grad(y, x, t, retain_graph=True)[0])(torch.ones_like(y))
    z = x * 1
    out, s = layer_norm(z, residual=torch.randn_like(z))
    s.add_(1)  # what backward would read
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


@pytest.mark.gpu
def test_saved_tensors_that_come_back_as_others(cuda_device):
    x = torch.randn(4, 16, device=cuda_device, requires_grad=True)
    w = torch.randn(16, device=cuda_device, requires_grad=True)
    want = torch.autograd.grad(layer_norm(x, w), (x, w), torch.ones_like(x))
    with torch.autograd.graph.save_on_cpu():
        y = layer_norm(x, w)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, (x, w), torch.ones_like(x)), want))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.t().contiguous().t()):
        y = layer_norm(x, w)
    got = torch.autograd.grad(y, (x, w), torch.ones_like(x))
    assert all(torch.allclose(a, b, atol=1e-5) for a, b in zip(got, want))
    for change in (lambda t: t.double(), lambda t: t[:2], lambda t: t.cpu()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
            y = layer_norm(x, w)
        with pytest.raises(RuntimeError, match="layer_norm: a (tensor saved for the backward pass|dense CUDA tensor)"):
            torch.autograd.grad(y, (x, w), torch.ones_like(x))


@pytest.mark.gpu
def test_results_do_not_depend_on_the_run(cuda_device):
    t = _inputs(2500, 1024, torch.bfloat16, torch.float32, torch.bfloat16, torch.float32, cuda_device)
    first = _call(t, None)
    for _ in range(3):
        again = _call(t, None)
        assert all(torch.equal(a, b) for a, b in zip(first[0] + first[1], again[0] + again[1]))


@pytest.mark.gpu
def test_captured_replayed_and_on_another_stream(cuda_device):
    t = _inputs(70, 1000, torch.bfloat16, torch.float32, torch.bfloat16, torch.float32, cuda_device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            out = _call(t, None)
    torch.cuda.current_stream().wait_stream(side)
    _check(t, None, *out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _call(t, None)
    other = _inputs(70, 1000, torch.bfloat16, torch.float32, torch.bfloat16, torch.float32, cuda_device, seed=8)
    with torch.no_grad():
        for k, v in other.items():
            t[k].copy_(v)
    graph.replay()
    _check(t, None, *out)


@pytest.fixture
def emptied():
    """What a test of several GB leaves in torch's cache is given back behind it: other tests count on what is free."""
    yield
    torch.cuda.empty_cache()


@pytest.mark.gpu
def test_places_beyond_32_bits(emptied, cuda_device):
    rows, cols = 70000, 32768
    x = torch.empty(rows, cols, device=cuda_device, dtype=torch.bfloat16)
    x.normal_(generator=torch.Generator(device=cuda_device).manual_seed(2))
    x.requires_grad_()
    y = layer_norm(x)
    ends = torch.tensor([0, 65535, 65536, rows - 1], device=cuda_device)
    part = x.detach()[ends].requires_grad_()
    want = layer_norm(part)
    assert torch.equal(y.detach()[ends], want.detach())
    g = torch.autograd.grad(y, x, y.detach())[0]
    assert torch.equal(g[ends], torch.autograd.grad(want, part, want.detach())[0])


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [17, 31, 33, 63, 65, 127, 129, 253, 259, 511, 513, 1023, 1025, 1535, 1537, 2047, 2049, 4095, 4099, 6143, 6145, 8191, 8209])
@pytest.mark.parametrize("dtype,stream", [(torch.float32, None), (torch.bfloat16, torch.float32), (torch.float16, torch.float16)])
def test_rows_that_begin_anywhere(cuda_device, cols, dtype, stream):
    # more rows than blocks have at once, where the row is short; a few more than one else
    t = _inputs(5000 if cols < 300 else 600, cols, dtype, stream, dtype, torch.float32, cuda_device, seed=cols)
    _check(t, None, *_call(t, None))


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [8200, 8196, 12290, 24584, 40961])
def test_rows_that_are_long(cuda_device, cols):
    # more rows than blocks, and than the sums' parts take at a time
    t = _inputs(650, cols, torch.bfloat16, torch.float32, torch.bfloat16, torch.float32, cuda_device, seed=cols)
    _check(t, None, *_call(t, None))
    t = _inputs(5, cols, torch.bfloat16, None, torch.float32, None, cuda_device, seed=cols)
    _check(t, torch.float32, *_call(t, torch.float32))


@pytest.mark.gpu
def test_rows_whose_numbers_32_bits_cannot_count_are_refused(cuda_device):
    one = torch.ones(1, device=cuda_device, dtype=torch.bfloat16)
    for shape in ((1, 2 ** 31 - 256), (2 ** 31, 1), (2, 2 ** 31)):
        with pytest.raises(RuntimeError, match="layer_norm: at most"):
            layer_norm(one.expand(shape))


@pytest.mark.parametrize("device", DEVICES)
def test_one_tensor_twice(device):
    x = torch.randn(5, 24, device=device, generator=torch.Generator(device=device).manual_seed(1))
    w = torch.randn(24, device=device, generator=torch.Generator(device=device).manual_seed(2))
    ds, dy = torch.randn_like(x), torch.randn_like(x)

    def run(leaf, of):
        y, s = of(leaf)
        torch.autograd.backward((y, s), (dy.to(y.dtype), ds.to(s.dtype)))
        return y.detach().double(), s.detach().double(), leaf.grad.double()

    def plain(t):
        s = t + t
        return torch.nn.functional.layer_norm(s, (24,), w.double(), w.double()), s

    got = run(x.clone().requires_grad_(), lambda t: layer_norm(t, w, w, residual=t))
    want = run(x.double().requires_grad_(), plain)
    for a, b in zip(got, want):
        # a few dozen roundings of terms a few times the result's size
        assert torch.allclose(a, b, rtol=64 * 2.0 ** -24, atol=64 * 2.0 ** -24 * b.abs().max().item())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype,stream", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("shape", [(24,), (6, 24), (2, 3, 24), (2, 3, 4, 24)])
@pytest.mark.parametrize("only", [None, 0, 1])
def test_gradients_of_leaves_have_memory_of_their_own(device, dtype, stream, shape, only):
    gen = torch.Generator().manual_seed(4)
    x, r = torch.randn(shape, generator=gen).to(device, dtype).requires_grad_(), torch.randn(shape, generator=gen).to(device, stream).requires_grad_()
    given = [torch.randn(shape, generator=gen).to(device, t) for t in (dtype, stream)]
    kept = [g.clone() for g in given]
    for turn in (1, 2):
        out = layer_norm(x, residual=r)
        (dx, dr) = torch.autograd.grad([o for i, o in enumerate(out) if only in (None, i)], (x, r), [g for i, g in enumerate(given) if only in (None, i)], retain_graph=True)
        torch.autograd.backward([o for i, o in enumerate(out) if only in (None, i)], [g for i, g in enumerate(given) if only in (None, i)])
        # (the same numbers twice are twice these, exactly)
        assert torch.equal(x.grad, turn * dx) and torch.equal(r.grad, turn * dr) and out[0].shape == out[1].shape == shape
        assert x.grad.untyped_storage().data_ptr() != r.grad.untyped_storage().data_ptr()
    assert all(torch.equal(a, b) for a, b in zip(given, kept))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype,stream", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float16, torch.float16)])
def test_one_of_the_results_alone(device, dtype, stream):
    gen = torch.Generator().manual_seed(9)
    x, r, w, b = (torch.randn(s, generator=gen).to(device, t).requires_grad_() for s, t in (((3, 5, 40), dtype), ((3, 5, 40), stream), ((40,), torch.float32), ((40,), torch.float32)))
    dy, ds = torch.randn(3, 5, 40, generator=gen).to(device, dtype), torch.randn(3, 5, 40, generator=gen).to(device, stream)
    leaves = (x, w, b, r)
    none_s = torch.autograd.grad(layer_norm(x, w, b, residual=r), leaves, (dy, torch.zeros_like(ds)))
    got = torch.autograd.grad(layer_norm(x, w, b, residual=r)[0], leaves, dy)
    assert all(torch.equal(a, c) for a, c in zip(got, none_s))
    got = torch.autograd.grad(layer_norm(x, w, b, residual=r)[1], leaves, ds)
    assert torch.equal(got[0], ds.to(dtype)) and torch.equal(got[3], ds) and float(got[1].abs().sum()) == float(got[2].abs().sum()) == 0
    assert [g.dtype for g in got] == [t.dtype for t in leaves] and [g.shape for g in got] == [t.shape for t in leaves]
    got = torch.autograd.grad(layer_norm(x, w, b, residual=r.detach())[1], leaves[:3], ds)
    assert torch.equal(got[0], ds.to(dtype))


@pytest.mark.gpu
def test_gradients_that_there_are_not_take_no_memory(cuda_device):
    x = torch.randn(2048, 1024, device=cuda_device, dtype=torch.bfloat16, requires_grad=True)
    r = torch.randn(2048, 1024, device=cuda_device, requires_grad=True)
    for which, most in ((0, 2048 * 1024 * 6), (1, 2048 * 1024 * 2)):  # dx and the residual's; of the sum alone dx is ds in another type
        out = layer_norm(x, residual=r)[which]
        given = torch.randn_like(out)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        grads = torch.autograd.grad(out, (x, r), given)
        assert torch.cuda.max_memory_allocated() - before <= most
        del out, grads


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("shape", [(16,), (5, 16), (2, 3, 16), (2, 2, 3, 16)])
def test_tensors_that_are_changed_in_place(device, shape):
    for call, changed in ((lambda x: (layer_norm(x),), lambda x, out: x), (lambda x: layer_norm(x, residual=x), lambda x, out: out[1])):
        x = torch.randn(shape, device=device, requires_grad=True) * 2
        out = call(x)
        changed(x, out).add_(1)  # what backward would read
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out[0].sum().backward()
        x = torch.randn(shape, device=device, requires_grad=True) * 2
        out = call(x)[0]
        out.mul_(2)  # what it would not
        out.sum().backward()
