"""What the decoder-block operators save for their backward pass, through hooks that bring it back otherwise."""
import pytest
import torch

from mccl_b200.ops import checkpoint
from mccl_b200.ops.gated import gated_feed_forward
from mccl_b200.ops.heads import norm_rotate, norm_rotate_packed, rotary_table

pytestmark = pytest.mark.gpu


def _rand(*shape, dtype=torch.float32, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


def _gated(dtype, eight):
    args = [_rand(70, 72, dtype=dtype), _rand(130, 72, dtype=dtype, seed=1), _rand(130, 72, dtype=dtype, seed=2), _rand(72, 130, dtype=dtype, seed=3)]
    return args, lambda *a: (gated_feed_forward(*a, checkpoint=eight),)


def _linear(dtype, _):
    return [_rand(70, 72, dtype=dtype), _rand(130, 72, dtype=dtype, seed=1)], lambda *a: (checkpoint.linear(*a),)


def _heads(dtype, _):
    table, pos = rotary_table(64, 32, device="cuda"), torch.randint(0, 64, (2, 9), device="cuda")
    args = [_rand(2, 9, 4, 64, dtype=dtype), _rand(2, 9, 2, 64, dtype=dtype, seed=1), _rand(64, seed=2), _rand(64, seed=3)]
    return args, lambda *a: norm_rotate(*a, table, pos)


def _packed(dtype, _):
    table, pos = rotary_table(64, 32, device="cuda"), torch.randint(0, 64, (2, 9), device="cuda")
    args = [_rand(2, 9, 8 * 64, dtype=dtype), _rand(64, seed=2), _rand(64, seed=3)]
    return args, lambda *a: norm_rotate_packed(*a, table, pos, heads=4, kv_heads=2)


CALLS = [(_gated, torch.bfloat16, None), (_gated, torch.bfloat16, "int8"), (_gated, torch.float32, None), (_gated, torch.float32, "int8"),
         (_linear, torch.float32, None), (_heads, torch.bfloat16, None), (_packed, torch.bfloat16, None), (_packed, torch.float32, None)]


def _gradients(call, args, unpack):
    args = [a.detach().clone().requires_grad_() for a in args]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        out = call(*args)
    return torch.autograd.grad([o for o in out if o.requires_grad], args, [torch.ones_like(o) for o in out if o.requires_grad])


def _apart(t):  # every second number of twice as many
    big = torch.zeros(*t.shape[:-1], 2 * t.shape[-1], dtype=t.dtype, device=t.device)[..., ::2]
    return big.copy_(t)


def _shifted(t):  # one number further than an aligned start
    return torch.zeros(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape).copy_(t)


@pytest.mark.parametrize("how", [torch.clone, _apart, _shifted, lambda t: t.cpu().cuda()])
@pytest.mark.parametrize("make,dtype,eight", CALLS)
def test_other_memory_is_fine(make, dtype, eight, how):
    args, call = make(dtype, eight)
    want, got = _gradients(call, args, lambda t: t), _gradients(call, args, how)
    # another layout may have another split of a row over lanes, and so another order of its sums
    assert all(torch.equal(a, b) if make is _gated and dtype != torch.float32 else torch.allclose(a, b, rtol=2.0 ** -7 if dtype != torch.float32 else 1e-4, atol=1e-3)
               for a, b in zip(want, got))


def _longer(t):
    return torch.cat((t, t), 0)


@pytest.mark.parametrize("how", [lambda t: t.cpu(), lambda t: t[..., :-1], lambda t: t[:-1], _longer, lambda t: t.flatten()[:1], lambda t: t.double(),
                                 lambda t: t.to(torch.int16)])
@pytest.mark.parametrize("make,dtype,eight", CALLS[:4])
def test_another_tensor_is_refused(make, dtype, eight, how):
    args, call = make(dtype, eight)
    seen = []
    _gradients(call, args, lambda t: seen.append(t) or t)
    for i in range(len(seen)):
        at = iter(range(len(seen)))
        # (integers for an input that requires a gradient: torch refuses them before)
        with pytest.raises(RuntimeError, match="MCCL|Only Tensors of floating point"):
            _gradients(call, args, lambda t: how(t) if next(at) == i else t)


@pytest.mark.parametrize("how", [lambda t: t.cpu(), lambda t: t[..., :-1], lambda t: t.flatten()[:1], lambda t: t.to(torch.int16)])
@pytest.mark.parametrize("make,dtype,eight", CALLS[4:])
def test_all_of_them_others_is_refused(make, dtype, eight, how):
    args, call = make(dtype, eight)
    with pytest.raises(RuntimeError):
        _gradients(call, args, how)
