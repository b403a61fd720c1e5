"""GPT-2 on this package's layer norm and linear layers, trained with moments in 8 bits: the operators as they are used together."""
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from mccl_b200.models import gpt2_tiny
from mccl_b200.optim import FusedAdamW
from mccl_b200.utils.spawn import run_workers

ROOT = Path(__file__).resolve().parents[1]
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _both(device, dtype=torch.float32):
    torch.manual_seed(0)
    a, b = gpt2_tiny(), gpt2_tiny(fused=True)
    with torch.no_grad():  # biases and norms that are not where they start
        for p in a.parameters():
            if p.dim() == 1:
                p.add_(0.1 * torch.randn_like(p))
    b.load_state_dict(a.state_dict())
    return a.to(device, dtype), b.to(device, dtype)


def _batch(device, batch=2, tokens=33):
    ids = torch.randint(0, 1024, (batch, tokens), generator=torch.Generator().manual_seed(3)).to(device)
    return ids[:, :-1].contiguous(), ids[:, 1:].contiguous()


@pytest.mark.parametrize("device", DEVICES)
def test_the_same_model_in_fp32(device):
    a, b = _both(device)
    x, y = _batch(device)
    assert list(a.state_dict()) == list(b.state_dict())
    wanted, got = a(x), b(x)
    # some 40 operators one behind the other, each within a few hundred roundings of 2^-24 of what it adds up
    assert (got - wanted).norm() <= 40 * 300 * 2.0 ** -24 * wanted.norm()
    a(x, y).backward(), b(x, y).backward()
    for (name, p), q in zip(a.named_parameters(), b.parameters()):
        assert (q.grad - p.grad).norm() <= 100 * 300 * 2.0 ** -24 * p.grad.norm(), name


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("whole", [False, True])
def test_gradients_in_16_bits_are_as_near_as_the_stock_models(device, dtype, whole):
    a, b = _both(device)
    x, y = _batch(device)
    a(x, y).backward()
    want = [p.grad.clone() for p in a.parameters()]
    off = []
    for m in (a, b):
        m.zero_grad()
        if whole:  # a model of that type
            m = m.to(dtype)
            loss = m(x, y)
        else:
            with torch.autocast(device, dtype=dtype):
                loss = m(x, y)
        (loss * 64).backward()
        off.append([float((p.grad.float() / 64 - w).norm() / w.norm()) for p, w in zip(m.parameters(), want)])
    # Both round some thirty times to 2^-8 (2^-11) on the way to each gradient; the fused one, which keeps more of it in fp32, no more often.
    # Two such sums of roundings of either sign differ by half at most in all but rare cases; four times allowed for.
    for name, stock, own in zip((n for n, _ in a.named_parameters()), *off):
        assert own <= 4 * stock + 2.0 ** (-8 if dtype is torch.bfloat16 else -11), (name, stock, own)


@pytest.mark.parametrize("device", DEVICES)
def test_one_token_alone(device):
    a, b = _both(device)
    ids = torch.tensor([[5], [77]], device=device)
    with torch.no_grad():
        for dtype, near in ((torch.float32, 1e-4), (torch.bfloat16, 0.1)):
            a, b = a.to(dtype), b.to(dtype)
            assert (a(ids).float() - b(ids).float()).norm() <= near * a(ids).float().norm()


@pytest.mark.gpu
def test_its_kernels_run(cuda_device):
    import mccl_b200
    native = mccl_b200.require_native()
    _, b = _both(cuda_device)
    x, y = _batch(cuda_device)
    before = native._kernel_launches()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = b(x, y)
    # of each of four layers two norms and four linear layers, and the last norm
    assert native._kernel_launches() - before >= 4 * 6 + 1
    before = native._kernel_launches()
    loss.backward()
    assert native._kernel_launches() - before >= 4 * (2 * 2 + 4 * 3) + 2


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,bits", [(torch.float32, 8), (torch.bfloat16, 8), (torch.bfloat16, 32)])
def test_trains_with_moments_in_8_bits_or_a_16_bit_model(cuda_device, dtype, bits):
    _, m = _both(cuda_device, dtype)
    x, y = _batch(cuda_device)
    opt = FusedAdamW(m.parameters(), lr=1e-3, state_bits=bits)
    before = [p.detach().clone() for p in m.parameters()]
    for _ in range(3):
        opt.zero_grad()
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=dtype is torch.float32):
            loss = m(x, y)
        loss.backward()
        opt.step()
    assert torch.isfinite(loss)
    for (name, p), q in zip(m.named_parameters(), before):
        # three steps of at most lr each, and the decay, in the type's rounding
        if name != "wpe.weight" and name != "wte.weight":
            assert not torch.equal(p, q), name
        room = 3 * 1e-3 * (1.2 + 0.01 * q.abs().float().max()) + (2.0 ** -8 * q.abs().float().max() if dtype is torch.bfloat16 else 1e-6)
        assert (p.detach().float() - q.float()).abs().max() <= room, name


@pytest.mark.gpu
def test_a_captured_step_is_the_step(cuda_device):
    _, m = _both(cuda_device, torch.bfloat16)
    x, y = _batch(cuda_device)
    params = list(m.parameters())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = torch.autograd.grad(m(x, y), params)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(m(x, y), params)
    graph.replay()
    for (name, _), g, w in zip(m.named_parameters(), got, want):
        # (the embedding's gradient is torch's, whose sums have no fixed order)
        assert torch.equal(g, w) or "wte" in name or "wpe" in name, name


def _ddp(rank, ws):
    import torch
    from mccl_b200.models import gpt2_tiny
    from mccl_b200.optim import FusedAdamW
    from mccl_b200.parallel import wrap_ddp
    torch.manual_seed(1)
    m = gpt2_tiny(fused=True).to(device)
    on_cuda = device.type == "cuda"
    opt = FusedAdamW(m.parameters(), lr=1e-3, state_bits=8) if on_cuda else torch.optim.AdamW(m.parameters(), lr=1e-3)
    ddp = wrap_ddp(m, device_ids=[device.index] if on_cuda else None, **({"optimizer_in_backward": opt} if on_cuda else {}))
    ids = torch.randint(0, 1024, (2, 17), generator=torch.Generator().manual_seed(rank)).to(device)
    for _ in range(3):
        opt.zero_grad()
        with torch.autocast(device.type, dtype=torch.bfloat16):
            loss = ddp(ids[:, :-1].contiguous(), ids[:, 1:].contiguous())
        loss.backward()
        opt.step()
    assert torch.isfinite(loss)
    if on_cuda:
        return
    flat = torch.cat([p.detach().reshape(-1) for p in m.parameters()])
    other = flat.clone()
    dist.broadcast(other, 0)
    assert torch.equal(flat, other)


def test_two_cpu_ranks():
    run_workers(_ddp, 2, timeout=240)


@pytest.mark.gpu
def test_ddp_on_one_gpu_with_the_optimizer_in_backward():
    run_workers(_ddp, 1, device="cuda", timeout=240)


def _example(*more):
    r = subprocess.run([sys.executable, "examples/ddp_dummy_train.py", "--baseline", "--model", "gpt2-tiny", "--fused-blocks", "--steps", "3", "--warmup", "1",
                        "--batch-size", "2", *more], cwd=ROOT, env=dict(os.environ), capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and "avg_step" in r.stdout, r.stderr[-2000:]


def test_example_on_the_cpu():
    _example("--cpu")


@pytest.mark.gpu
def test_example_with_moments_in_8_bits():
    _example("--fused-optim", "--moment-bits", "8", "--fp16")


@pytest.mark.parametrize("args,what", [
    (["--cpu", "--model", "gpt2-tiny", "--moment-bits", "8"], "--moment-bits 8 is for"),
    (["--cpu", "--model", "gpt2-tiny", "--fused-optim", "--moment-bits", "8"], "--moment-bits 8 is for"),
    (["--cpu", "--model", "gated-tiny", "--fused-blocks"], "--fused-blocks is for"),
    (["--model", "mlp", "--fused-blocks"], "--fused-blocks is for")])
def test_example_refuses_flags_without_effect(args, what, monkeypatch, capsys):
    import runpy
    monkeypatch.setattr(sys, "argv", ["ddp_dummy_train.py", "--baseline", *args])
    with pytest.raises(SystemExit) as e:
        runpy.run_path(str(ROOT / "examples/ddp_dummy_train.py"), run_name="__main__")
    assert e.value.code == 2 and what in capsys.readouterr().err


@pytest.mark.parametrize("args,what", [
    (["--model", "gpt2-tiny", "--impl", "nccl", "--moment-bits", "8"], "--moment-bits 8 is for"),
    (["--model", "resnet50", "--moment-bits", "8"], "--moment-bits 8 is for"),
    (["--model", "resnet50", "--fused-blocks"], "--fused-blocks is for"),
    (["--model", "mlp", "--fused-blocks"], "--fused-blocks is for")])
def test_benchmark_refuses_flags_without_effect(args, what, capsys):
    from mccl_b200.bench.ddp import main
    with pytest.raises(SystemExit) as e:
        main(args)
    assert e.value.code == 2 and what in capsys.readouterr().err
