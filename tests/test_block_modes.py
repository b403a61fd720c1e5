"""The operators of a decoder block under modes that have to see what a call is made of: traces and counts are right."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils.flop_counter import FlopCounterMode

from mccl_b200.ops import checkpoint
from mccl_b200.ops.checkpoint import pack8, unpack8
from mccl_b200.ops.gated import gated_feed_forward
from mccl_b200.ops.heads import norm_rotate, norm_rotate_packed, rotary_table

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
U = 2.0 ** -24


def _gen(device):
    gen = torch.Generator().manual_seed(7)
    return lambda *s: torch.randn(*s, generator=gen).to(device)


def _gated(x, wg, wu, wd):
    g = x @ wg.T
    return (g * torch.sigmoid(g) * (x @ wu.T)) @ wd.T


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("pre_dispatch", [False, True])
def test_a_trace_of_the_gated_block_answers_for_other_inputs(device, pre_dispatch):
    rand = _gen(device)
    x, other, wg, wu, wd = rand(9, 24), rand(9, 24), rand(40, 24), rand(40, 24), rand(24, 40)
    traced = make_fx(lambda t: gated_feed_forward(t, wg, wu, wd), pre_dispatch=pre_dispatch)(x)
    want = _gated(*(t.double() for t in (other, wg, wu, wd)))
    # each product's terms round once and its sums once a term; two products of 24 and 40 terms, the gate within 2^-20
    g, u = other.abs().double() @ wg.abs().double().T, other.abs().double() @ wu.abs().double().T
    assert ((traced(other).double() - want).abs() <= (g * u) @ wd.abs().double().T * (2 * 26 + 42 + 32) * U).all()


@pytest.mark.parametrize("device", DEVICES)
def test_a_trace_of_a_training_step_answers_for_other_inputs(device):
    rand = _gen(device)
    x, other, wg, wu, wd, dy = rand(9, 24), rand(9, 24), rand(40, 24), rand(40, 24), rand(24, 40), rand(9, 24)

    def step(t):
        t = t.detach().requires_grad_()
        return torch.autograd.grad(gated_feed_forward(t, wg, wu, wd), t, dy)[0]

    traced = make_fx(step)(x)
    t = other.double().requires_grad_()
    (want,) = torch.autograd.grad(_gated(t, *(w.double() for w in (wg, wu, wd))), t, dy.double())
    # products of 40 and 24 terms of size one or so with weights of size one: gradients of size 40 to 100, each of whose roundings
    # is below 2^-24 of the sum of what it adds up, some thousand times the largest number
    assert (traced(other).double() - want).abs().max() <= 100 * 24 * 40 * U * want.abs().max()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("packed", [False, True])
def test_a_trace_of_the_heads_answers_for_other_inputs(device, packed):
    rand = _gen(device)
    w, table = [1 + 0.1 * rand(16) for _ in range(2)], rotary_table(32, 16, device=device)

    def call(t):
        if packed:
            return norm_rotate_packed(t, *w, table, heads=2, kv_heads=1)[:2]
        q, k = t.unflatten(-1, (4, 16))[:, :, :3].split((2, 1), 2)
        return norm_rotate(q, k, *w, table)

    x, other = rand(2, 5, 64), rand(2, 5, 64)
    got, want = make_fx(call)(x)(other), call(other)
    # the same formula: r within 16 roundings, products and the rotation's sum of two within 8
    assert all(((a - b).abs() <= 48 * U * 2 * b.abs().max()).all() for a, b in zip(got, want))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_trace_of_the_checkpoints_answers_for_other_inputs(device, dtype):
    rand = _gen(device)
    x, other = rand(7, 100).to(dtype), rand(7, 100).to(dtype)
    assert torch.equal(make_fx(lambda t: unpack8(pack8(t)))(x)(other), unpack8(pack8(other)))


@pytest.mark.parametrize("device", DEVICES)
def test_floating_point_operations_are_counted(device):
    rand = _gen(device)
    x, wg, wu, wd = rand(9, 24), rand(40, 24), rand(40, 24), rand(24, 40)
    with FlopCounterMode(display=False) as count:
        gated_feed_forward(x, wg, wu, wd)
        checkpoint.linear(x, wg)
    assert count.get_total_flops() == 2 * 9 * 24 * 40 * 4
    args = [t.requires_grad_() for t in (x, wg, wu, wd)]
    with FlopCounterMode(display=False) as count:
        gated_feed_forward(*args).sum().backward()
    assert count.get_total_flops() == 2 * 9 * 24 * 40 * 9


@pytest.mark.gpu
def test_outside_of_modes_the_kernels_answer():
    import mccl_b200
    native = mccl_b200.require_native()
    rand = _gen("cuda")
    x, w, d = rand(9, 24).bfloat16(), rand(40, 24).bfloat16(), rand(24, 40).bfloat16()
    with FlopCounterMode(display=False):
        before = native._kernel_launches()
        gated_feed_forward(x, w, w, d), unpack8(pack8(x))
        assert native._kernel_launches() == before
    with torch.device("cuda"):  # a mode of functions, not of operators
        gated_feed_forward(x, w, w, d), unpack8(pack8(x))
    assert native._kernel_launches() >= before + 4


@pytest.mark.gpu
@pytest.mark.parametrize("pre_dispatch", [False, True])
def test_a_trace_of_a_backward_pass_alone_is_refused(pre_dispatch):
    rand = _gen("cuda")
    x, w, d, dy = rand(9, 24).requires_grad_(), rand(40, 24), rand(24, 40), rand(9, 24)
    y = gated_feed_forward(x, w, w, d)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(lambda t: torch.autograd.grad(y, x, t, retain_graph=True)[0], pre_dispatch=pre_dispatch)(dy)
    q, ones, table = rand(1, 5, 2, 16).requires_grad_(), torch.ones(16, device="cuda"), rotary_table(8, 16, device="cuda")
    r, _ = norm_rotate(q, q, ones, ones, table)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(lambda t: torch.autograd.grad(r, q, t, retain_graph=True)[0], pre_dispatch=pre_dispatch)(torch.ones_like(r))
    with FlopCounterMode(display=False):  # what a mode cannot see does no harm elsewhere
        torch.autograd.grad(y, x, dy)
