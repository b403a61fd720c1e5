"""Norms and rotation of queries and keys against the formulas in 64 bits."""
import math

import pytest
import torch

from mccl_b200.ops.heads import norm_rotate, norm_rotate_packed, rotary_table

U = 2.0 ** -24
ROUNDOFF = {torch.float32: U, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
EPS = 1e-6


def _split(x, rotary, near):
    return ((x[..., 0:rotary:2], x[..., 1:rotary:2]) if near else (x[..., :rotary // 2], x[..., rotary // 2:rotary])) + (x[..., rotary:],)


def _merge(a, b, rest, near):
    return torch.cat((torch.stack((a, b), -1).flatten(-2) if near else torch.cat((a, b), -1), rest), -1)


def _angles(table, positions, batch):
    cs = table.double()[positions].expand(batch, -1, -1, -1) if positions.dim() == 2 else table.double()[positions][None].expand(batch, -1, -1, -1)
    return cs[:, :, None, 0], cs[:, :, None, 1]


def _value(x, w, cos, sin, near, rotary):
    n = x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * w
    a, b, rest = _split(n, rotary, near)
    size = _merge((a * cos).abs() + (b * sin).abs(), (b * cos).abs() + (a * sin).abs(), rest.abs(), near)
    return _merge(a * cos - b * sin, b * cos + a * sin, rest, near), size


def _gradient(dy, x, w, cos, sin, near, rotary):
    """The formulas' gradients, and the sums of the absolute values of what they add up."""
    r = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
    a, b, rest = _split(dy, rotary, near)
    dn = _merge(a * cos + b * sin, b * cos - a * sin, rest, near)
    size = _merge((a * cos).abs() + (b * sin).abs(), (b * cos).abs() + (a * sin).abs(), rest.abs(), near)
    dx = r * (dn * w - x * r * r * (dn * w * x).mean(-1, keepdim=True))
    dx_size = r * (size * w.abs() + x.abs() * r * r * (size * w.abs() * x.abs()).mean(-1, keepdim=True))
    return dx, (dn * x * r).sum((0, 1, 2)), dx_size, (size * x.abs() * r).sum((0, 1, 2))


def _near(got, want, size, steps):
    """`steps` roundings of 2^-24 of what is added up, and the result's own."""
    off = (got.detach().double() - want).abs()
    # (a result a rounding away from the exact one may round to the next number)
    return (off <= size * steps * U * (1 + ROUNDOFF[got.dtype]) + want.abs() * ROUNDOFF[got.dtype] + SMALLEST[got.dtype]).all()


# Sum of the squares: 16 in a lane, at most 5 between lanes, mean and eps: 23, halved by the root; the root's own 4: r is within 16.
# Forward: r, two products, and the rotation's product and sum: 21.  dx: dn 2; two sums of 16 + 5 products of three; three times r:
# below 80.  dw: dn 2, x r 17, product 1, heads / parts in a lane, 5 + 8 in a block, up to 900 / 32 + 12 over the blocks.
FORWARD, DX, DW = 24, 80, 160


def _case(batch, tokens, heads, kv, dim, rotary, near, dtype, packed, weights=torch.float32, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    t = {"w": [(1 + 0.3 * rand(dim)).to(weights) for _ in range(2)], "table": rotary_table(tokens + 300, rotary, device="cuda"),
         "positions": torch.randint(0, tokens + 300, (batch, tokens), generator=gen, device="cuda")}
    if packed:
        t["qkv"] = rand(batch, tokens, (heads + 2 * kv) * dim).to(dtype)
        rows = t["qkv"].unflatten(-1, (-1, dim))
        t["x"] = [rows[:, :, :heads], rows[:, :, heads:heads + kv], rows[:, :, heads + kv:]]
    else:
        t["x"] = [rand(batch, tokens, n, dim).to(dtype) for n in (heads, kv)]
    t["dy"] = [rand(batch, tokens, n, dim).to(dtype) for n in (heads, kv, kv)]
    return t


CASES = [
    # batch, tokens, heads, kv heads, dim, rotary, neighbours
    (1, 1, 1, 1, 64, 64, False), (2, 3, 5, 2, 64, 64, True), (1, 130, 4, 4, 128, 128, False), (3, 17, 6, 3, 80, 32, True),
    (3, 17, 6, 3, 80, 32, False), (2, 9, 3, 1, 96, 48, False), (2, 9, 3, 1, 96, 48, True), (1, 40, 2, 2, 31, 30, False),
    (1, 40, 2, 2, 31, 14, True), (2, 5, 1, 1, 1, 0, False), (2, 5, 2, 1, 2, 2, True), (1, 33, 3, 3, 256, 256, False), (1, 33, 3, 1, 512, 256, True),
    (1, 7, 2, 2, 511, 400, False), (2, 11, 4, 2, 100, 50, False), (2, 11, 4, 2, 100, 100, True), (1, 1000, 16, 4, 64, 32, False),
    (5, 1, 32, 8, 128, 128, True), (1, 21, 2, 1, 48, 0, False), (1, 300, 7, 7, 32, 24, False), (2, 6, 2, 2, 300, 8, True),
    (1, 9, 2, 1, 264, 264, False), (1, 9, 2, 1, 264, 264, True), (3, 500, 24, 24, 64, 64, False), (1, 3000, 2, 1, 128, 128, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("batch,tokens,heads,kv,dim,rotary,near", CASES)
def test_matches_64_bits(batch, tokens, heads, kv, dim, rotary, near, dtype, packed):
    t = _case(batch, tokens, heads, kv, dim, rotary, near, dtype, packed)
    w = [x.requires_grad_() for x in t["w"]]
    if packed:
        qkv = t["qkv"].requires_grad_()
        q, k, v = norm_rotate_packed(qkv, *w, t["table"], t["positions"], heads=heads, kv_heads=kv, interleaved=near)
        assert torch.equal(v, t["x"][2]) and v.data_ptr() == t["x"][2].data_ptr()
        grad, *dw = torch.autograd.grad((q, k, v), (qkv, *w), t["dy"])
        dx = grad.unflatten(-1, (-1, dim)).split((heads, kv, kv), 2)
        assert torch.equal(dx[2], t["dy"][2])
    else:
        x = [y.requires_grad_() for y in t["x"]]
        q, k = norm_rotate(*x, *w, t["table"], t["positions"], interleaved=near)
        *dx, dw0, dw1 = torch.autograd.grad((q, k), (*x, *w), t["dy"][:2])
        dw = [dw0, dw1]
    cos, sin = _angles(t["table"], t["positions"], batch)
    for i, got in enumerate((q, k)):
        x, wi, dy = t["x"][i].detach().double(), w[i].detach().double(), t["dy"][i].double()
        assert got.is_contiguous() and got.dtype == dtype
        assert _near(got, *_value(x, wi, cos, sin, near, rotary), FORWARD)
        want_dx, want_dw, dx_size, dw_size = _gradient(dy, x, wi, cos, sin, near, rotary)
        assert _near(dx[i], want_dx, dx_size, DX)
        assert dw[i].dtype == torch.float32 and _near(dw[i], want_dw, dw_size, DW)
    with torch.no_grad():  # serving: the same numbers
        again = (norm_rotate_packed(t["qkv"], *w, t["table"], t["positions"], heads=heads, kv_heads=kv, interleaved=near)[:2] if packed
                 else norm_rotate(*t["x"], *w, t["table"], t["positions"], interleaved=near))
    assert torch.equal(again[0], q) and torch.equal(again[1], k)


@pytest.mark.gpu
def test_gradient_against_differences():
    batch, tokens, heads, kv, dim, rotary, near = 2, 7, 3, 1, 40, 24, False
    t = _case(batch, tokens, heads, kv, dim, rotary, near, torch.float32, False, seed=3)
    x, w = [y.requires_grad_() for y in t["x"]], [y.requires_grad_() for y in t["w"]]
    q, k = norm_rotate(*x, *w, t["table"], t["positions"], interleaved=near)
    grads = torch.autograd.grad((q, k), (*x, *w), t["dy"][:2])
    cos, sin = _angles(t["table"], t["positions"], batch)

    def loss(xs, ws):
        return sum((_value(a, b, cos, sin, near, rotary)[0] * dy.double()).sum() for a, b, dy in zip(xs, ws, t["dy"]))

    at = [y.detach().double() for y in (*x, *w)]
    for i, g in enumerate(grads):
        v = torch.randn(at[i].shape, dtype=torch.double, device="cuda", generator=torch.Generator(device="cuda").manual_seed(i))
        up, down = list(at), list(at)
        h = 1e-5
        up[i], down[i] = at[i] + h * v, at[i] - h * v
        slope = (loss(up[:2], up[2:]) - loss(down[:2], down[2:])) / (2 * h)
        # truncation (h^2 times third derivatives of order one over some 500 numbers) and cancellation (2^-53 |loss| / h) are below
        # 1e-6; the gradient itself is fp32: its size times the steps above
        bound = 1e-6 + (g.double().abs() * v.abs()).sum() * 4 * max(DX, DW) * U + v.abs().sum() * 40 * U
        assert abs((g.double() * v).sum() - slope) <= bound


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_layouts_give_the_same_numbers(dtype):
    t = _case(2, 19, 4, 2, 64, 64, False, dtype, False)
    q, k = t["x"]
    want = norm_rotate(q, k, *t["w"], t["table"], t["positions"])

    def other(x, how):
        if how == "heads first":
            return x.transpose(1, 2).contiguous().transpose(1, 2)
        if how == "odd start":
            wide = torch.zeros(*x.shape[:3], x.shape[3] + 3, dtype=dtype, device="cuda")[..., 1:x.shape[3] + 1]
            return wide.copy_(x)
        if how == "numbers apart":
            return torch.stack((x, x), -1)[..., 0]
        return x.flatten(2).clone().unflatten(2, x.shape[2:])

    # another split of the row over lanes may add its squares up in another order
    def alike(a, b):
        return ((a.double() - b.double()).abs() <= b.double().abs() * (2 * ROUNDOFF[dtype] + 2 * FORWARD * U) + 1e-6).all()

    for how in ("heads first", "odd start", "numbers apart", "copy"):
        got = norm_rotate(other(q, how), other(k, how), *t["w"], t["table"], t["positions"])
        assert alike(got[0], want[0]) and alike(got[1], want[1]), how
    for pos in (t["positions"].int(), t["positions"].t().contiguous().t()):
        got = norm_rotate(q, k, *t["w"], t["table"], pos)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    line = torch.arange(19, device="cuda")
    a = norm_rotate(q, k, *t["w"], t["table"])
    for pos in (line, line[None], line.expand(2, 19)):
        b = norm_rotate(q, k, *t["w"], t["table"], pos)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    same = norm_rotate(q[:1].expand(2, 19, 4, 64), k[:1, :, :1].expand(2, 19, 2, 64), *t["w"], t["table"])
    assert torch.equal(same[0][0], a[0][0]) and torch.equal(same[0][1], a[0][0]) and torch.equal(same[1][1, :, 1], a[1][0, :, 0])


@pytest.mark.gpu
def test_broadcast_and_missing_gradients_and_weights_of_the_type():
    t = _case(2, 19, 4, 2, 64, 64, False, torch.bfloat16, True, weights=torch.bfloat16)
    qkv, w = t["qkv"].requires_grad_(), [x.requires_grad_() for x in t["w"]]
    q, k, v = norm_rotate_packed(qkv, *w, t["table"], heads=4, kv_heads=2)
    one = torch.ones((), dtype=torch.bfloat16, device="cuda")
    a = torch.autograd.grad((q, k, v), (qkv, *w), [one.expand_as(x) for x in (q, k, v)], retain_graph=True)
    b = torch.autograd.grad((q, k, v), (qkv, *w), [torch.ones_like(x) for x in (q, k, v)], retain_graph=True)
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and a[1].dtype == torch.bfloat16
    only = torch.autograd.grad(k, (qkv, *w), torch.ones_like(k), retain_graph=True)
    assert not only[0][..., :4 * 64].any() and not only[0][..., 6 * 64:].any() and not only[1].any()
    assert torch.equal(only[0][..., 4 * 64:6 * 64], a[0][..., 4 * 64:6 * 64]) and torch.equal(only[2], a[2])
    (no_weights,) = torch.autograd.grad((q, k, v), qkv, [torch.ones_like(x) for x in (q, k, v)])
    assert torch.equal(no_weights, a[0])


@pytest.mark.gpu
def test_no_tokens_zero_rows_infinities_and_positions_outside():
    w = [torch.ones(64, device="cuda", requires_grad=True) for _ in range(2)]
    table = rotary_table(8, 32, device="cuda")
    q, k = torch.randn(2, 0, 3, 64, device="cuda", requires_grad=True), torch.randn(2, 0, 1, 64, device="cuda", requires_grad=True)
    a, b = norm_rotate(q, k, *w, table)
    assert a.shape == q.shape and b.shape == k.shape
    g = torch.autograd.grad((a, b), (q, k, *w), (a.detach(), b.detach()))
    assert g[0].shape == q.shape and not g[2].any() and not g[3].any()
    q, k = torch.randn(1, 5, 3, 64, device="cuda"), torch.randn(1, 5, 1, 64, device="cuda")
    q[0, 0] = 0
    q[0, 1, 0, 5] = float("inf")
    q[0, 2, 1, 40] = float("nan")
    pos = torch.tensor([0, 1, 2, 8, -1], device="cuda")
    q.requires_grad_(), k.requires_grad_()
    a, b = norm_rotate(q, k, *w, table, pos)
    assert not a[0, 0].any()
    assert torch.isnan(a[0, 1, 0, 5]) and torch.isfinite(a[0, 1, 1:]).all() and torch.isnan(a[0, 2, 1]).all() and torch.isfinite(a[0, 2, 2]).all()
    for t in (3, 4):
        assert torch.isnan(a[0, t, :, :32]).all() and torch.isfinite(a[0, t, :, 32:]).all() and torch.isnan(b[0, t, :, :32]).all()
    dq, dk = torch.autograd.grad((a, b), (q, k), (torch.ones_like(a), torch.ones_like(b)))
    assert torch.isfinite(dq[0, 0]).all() and torch.isfinite(dk[0, :3]).all() and torch.isnan(dk[0, 3:]).all()


@pytest.mark.gpu
def test_far_rows():
    # element offsets beyond 31 bits: queries 70000 elements a token apart
    tokens, dim = 40000, 64
    buf = torch.empty(tokens * 70000, dtype=torch.bfloat16, device="cuda")
    q = buf.as_strided((1, tokens, 1, dim), (buf.numel(), 70000, dim, 1))
    near = torch.randn(1, tokens, 1, dim, device="cuda").bfloat16()
    q.copy_(near)
    w, table = torch.ones(dim, device="cuda"), rotary_table(tokens, dim, device="cuda")
    a, _ = norm_rotate(q, near, w, w, table)
    b, _ = norm_rotate(near, near, w, w, table)
    assert torch.equal(a, b)


@pytest.mark.gpu
def test_streams_graphs_and_double_backward():
    t = _case(2, 50, 4, 2, 64, 64, False, torch.bfloat16, True)
    args = (t["qkv"], *t["w"], t["table"])
    want = norm_rotate_packed(*args, heads=4, kv_heads=2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = norm_rotate_packed(*args, heads=4, kv_heads=2)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = norm_rotate_packed(*args, heads=4, kv_heads=2)
    graph.replay()
    assert torch.equal(again[1], want[1])
    qkv = t["qkv"].requires_grad_()
    q, _, _ = norm_rotate_packed(qkv, *t["w"], t["table"], heads=4, kv_heads=2)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(q.float().sum(), qkv, create_graph=True)


@pytest.mark.gpu
def test_refusals():
    q, k, w = (torch.zeros(2, 3, 4, 64, device="cuda"), torch.zeros(2, 3, 2, 64, device="cuda"), torch.ones(64, device="cuda"))
    table, pos = rotary_table(16, 64, device="cuda"), torch.zeros(2, 3, dtype=torch.long, device="cuda")
    norm_rotate(q, k, w, w, table, pos)
    bad = [
        (q[0], k, w, w, table, pos), (q, k[:1], w, w, table, pos), (q, k[..., :32], w, w, table, pos), (q, k.half(), w, w, table, pos),
        (q.double(), k.double(), w, w, table, pos), (q, k.cpu(), w, w, table, pos), (q, k, w[:32], w, table, pos), (q, k, w.half(), w, table, pos),
        (q, k, w, w.cpu(), table, pos), (q, k, w, w, table.half(), pos), (q, k, w, w, table[:, :1], pos), (q, k, w, w, table.cpu(), pos),
        (q, k, w, w, rotary_table(16, 66, device="cuda"), pos), (q, k, w, w, table, pos.float()), (q, k, w, w, table, pos[:, :2]),
        (q, k, w, w, table, pos.cpu()), (q[:, :, :0], k, w, w, table, pos), (torch.zeros(1, 1, 1, 600, device="cuda"),) * 2 + (w, w, table, None),
    ]
    for args in bad:
        with pytest.raises(RuntimeError, match="MCCL"):
            norm_rotate(*args)
    for eps in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(RuntimeError, match="eps"):
            norm_rotate(q, k, w, w, table, pos, eps=eps)
    for heads, kv in ((4, 3), (0, 1), (1, 0), (-2, 1)):
        with pytest.raises(RuntimeError, match="MCCL"):
            norm_rotate_packed(torch.zeros(1, 2, 8 * 64, device="cuda"), w, w, table, heads=heads, kv_heads=kv)
    with pytest.raises(RuntimeError, match="transforms"):
        torch.func.vmap(lambda a: norm_rotate(a, a, w, w, table)[0])(torch.zeros(2, 1, 3, 4, 64, device="cuda"))


@pytest.mark.gpu
def test_tracing_is_refused():
    q, w, table = torch.zeros(1, 3, 2, 64, device="cuda"), torch.ones(64, device="cuda"), rotary_table(4, 64, device="cuda")
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda a: norm_rotate(a, a, w, w, table)[0], (q,))


@pytest.mark.parametrize("near", [False, True])
def test_cpu_form_and_its_gradient(near):
    torch.manual_seed(0)
    table = rotary_table(32, 12)
    assert torch.allclose(table[5, 0], torch.cos(5 * 10000.0 ** (-torch.arange(0, 12, 2, dtype=torch.double) / 12)).float())
    qkv = torch.randn(2, 5, 8 * 20, dtype=torch.float32, requires_grad=True)
    w = [torch.rand(20, requires_grad=True) for _ in range(2)]
    pos = torch.randint(0, 32, (2, 5))
    q, k, v = norm_rotate_packed(qkv, *w, table, pos, heads=4, kv_heads=2, interleaved=near)
    dy = [torch.randn_like(x) for x in (q, k, v)]
    grad, dwq, dwk = torch.autograd.grad((q, k, v), (qkv, *w), dy)
    cs = table.double()[pos]
    cos, sin = cs[:, :, None, 0], cs[:, :, None, 1]
    rows = qkv.detach().double().unflatten(-1, (-1, 20))
    for got, x, wi, d, dwi, at in ((q, rows[:, :, :4], w[0], dy[0], dwq, 0), (k, rows[:, :, 4:6], w[1], dy[1], dwk, 4)):
        want, size = _value(x, wi.detach().double(), cos, sin, near, 12)
        assert _near(got, want, size, FORWARD + 20)
        dx, dw, dx_size, dw_size = _gradient(d.double(), x, wi.detach().double(), cos, sin, near, 12)
        # (torch's own order of the backward pass: a few roundings more)
        assert _near(grad.unflatten(-1, (-1, 20))[:, :, at:at + x.shape[2]], dx, dx_size, 2 * DX)
        assert _near(dwi, dw, dw_size, DW)
    with pytest.raises(ValueError):
        norm_rotate_packed(qkv, *w, table, heads=3, kv_heads=2)
    with pytest.raises(ValueError):
        rotary_table(4, 3)
    assert math.isnan(norm_rotate(rows[:1, :1].float(), rows[:1, :1].float(), *w, table, torch.tensor([99]))[0].detach().sum())


def test_the_cpu_form_refuses_what_the_kernels_refuse():
    q, k, w = torch.zeros(2, 3, 4, 64), torch.zeros(2, 3, 2, 64), torch.ones(64)
    table, pos = rotary_table(16, 64), torch.zeros(2, 3, dtype=torch.long)
    norm_rotate(q, k, w, w, table, pos), norm_rotate(q, k, w, w, table, pos[0].int()), norm_rotate(q.half(), k.half(), w.half(), w.half(), table, pos[:1])
    bad = [
        (q[0], k, w, w, table, pos), (q, k[:1], w, w, table, pos), (q, k[..., :32], w, w, table, pos), (q, k.half(), w, w, table, pos),
        (q.double(), k.double(), w, w, table, pos), (q, k, w[:32], w, table, pos), (q, k, w[:1], w[:1], table, pos), (q, k, w, w.half(), table, pos),
        (q, k, w.half(), w.half(), table, pos), (q, k, w, w, table.half(), pos), (q, k, w, w, table.bfloat16(), pos), (q, k, w, w, table.double(), pos),
        (q, k, w, w, table[:, :1], pos), (q, k, w, w, table.clone().requires_grad_(), pos), (q, k, w, w, rotary_table(16, 66), pos),
        (q, k, w, w, table, pos.float()), (q, k, w, w, table, pos[:, :2]), (q, k, w, w, table, pos[:, 0]), (q[:, :, :0], k, w, w, table, pos),
        (torch.zeros(1, 1, 1, 600),) * 2 + (torch.ones(600),) * 2 + (table, None), (torch.zeros(1, 1, 1, 65),) * 2 + (torch.ones(65),) * 2 + (rotary_table(4, 128), None),
    ]
    for args in bad:
        with pytest.raises(ValueError, match="norm_rotate"):
            norm_rotate(*args)
    for eps in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="eps"):
            norm_rotate(q, k, w, w, table, pos, eps=eps)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_an_empty_table_has_no_position(device):
    x, w = torch.ones(1, 2, 1, 8, device=device), torch.ones(8, device=device)
    for pos in (None, torch.tensor([0, 5], device=device)):
        y = norm_rotate(x, x, w, w, rotary_table(0, 4, device=device), pos)[0]
        assert torch.isnan(y[..., :4]).all() and torch.isfinite(y[..., 4:]).all()
