"""The decoder of gated blocks: training, data-parallel training and decoding on the operators."""
import json
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import mccl_b200
from mccl_b200.models import GatedDecoder, gated_tiny
from mccl_b200.models.gated import GatedBlock

ROOT = Path(__file__).resolve().parents[1]
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _batch(device, batch=2, tokens=33):
    ids = torch.randint(0, 1024, (batch, tokens), generator=torch.Generator().manual_seed(3)).to(device)
    return ids[:, :-1], ids[:, 1:]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_learns_one_batch(checkpoint, device):
    torch.manual_seed(0)
    model = gated_tiny(checkpoint=checkpoint).to(device)
    x, y = _batch(device)
    opt = torch.optim.AdamW(model.parameters(), lr=3e-3)
    losses = []
    for _ in range(12):
        opt.zero_grad()
        loss = model(x, y)
        loss.backward()
        opt.step()
        losses.append(loss.item())
    assert losses[0] > 6.5 and losses[-1] < losses[0] - 2


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_gradients_under_autocast(checkpoint, dtype, device):
    torch.manual_seed(0)
    model = gated_tiny(checkpoint=checkpoint).to(device)
    x, y = _batch(device)
    model(x, y).backward()
    want = [p.grad for p in model.parameters()]
    model.zero_grad()
    with torch.autocast(device, dtype=dtype):
        loss = model(x, y)
    (loss * 256).backward()
    for (name, p), w in zip(model.named_parameters(), want):
        # some thirty roundings to 2^-8 (2^-11) one behind the other, of either sign; codes of 8 bits in both or in neither
        assert p.grad.dtype == torch.float32 and (p.grad / 256 - w).norm() <= (0.25 if dtype == torch.bfloat16 else 0.06) * w.norm(), name


@pytest.mark.parametrize("device", DEVICES)
def test_decoding_with_a_cache_is_the_whole_sequence_again(device):
    torch.manual_seed(1)
    model = gated_tiny().to(device)
    start = _batch(device, 3, 9)[0]
    got = model.generate(start, 5)
    want = start
    with torch.no_grad():
        for _ in range(5):
            want = torch.cat((want, model(want)[:, -1:].argmax(-1)), 1)
    assert torch.equal(got, want)
    with pytest.raises(ValueError, match="max_seq"):
        model.generate(start, 121)
    with pytest.raises(ValueError, match="max_seq"):
        model(torch.zeros(1, 129, dtype=torch.long, device=device))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float64])
@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_a_model_of_another_type(checkpoint, dtype, device):
    torch.manual_seed(4)
    model = gated_tiny(checkpoint=checkpoint)
    table, (x, y) = model.table.clone(), _batch(device)
    with torch.no_grad():
        want = model.to(device)(x)
    model = model.to(dtype)
    assert model.table.dtype == torch.float32 and torch.equal(model.table.cpu(), table) and "table" not in model.state_dict()
    assert model.table.device == model.wte.weight.device and torch.equal(model.cpu().float().table, table)
    if dtype == torch.float64:  # no type of the operators
        return
    model = model.to(device, dtype)
    logits = model(x)
    # some thirty roundings one behind the other, of either sign
    assert logits.dtype == dtype and (logits.float() - want).norm() <= (0.1 if dtype == torch.bfloat16 else 0.02) * want.norm()
    model(x, y).backward()
    assert all(p.grad.dtype == dtype and torch.isfinite(p.grad).all() for p in model.parameters())
    got = model.generate(x[:, :9], 3)
    assert got.shape == (2, 12) and torch.equal(got[:, :9], x[:, :9])


@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_projections_are_called_as_layers(checkpoint):
    torch.manual_seed(5)
    model, seen = gated_tiny(checkpoint=checkpoint), []
    block = model.blocks[0]
    for name in ("qkv", "proj"):
        getattr(block, name).register_forward_hook(lambda *a, name=name: seen.append(name))
    x, _ = _batch("cpu")
    model(x)
    assert seen == ["qkv", "proj"]

    class Twice(torch.nn.Module):
        def __init__(self, layer):
            super().__init__()
            self.layer, self.weight = layer, layer.weight

        def forward(self, t):
            return 2 * self.layer(t)

    with torch.no_grad():
        for b in model.blocks:
            b.proj = Twice(b.proj)
        replaced = model(x)
        for b in model.blocks:
            b.proj = b.proj.layer
            b.proj.weight.mul_(2)
        assert torch.equal(model(x), replaced)
    assert gated_tiny(checkpoint="int8").state_dict().keys() == gated_tiny().state_dict().keys()


def test_refusals():
    with pytest.raises(ValueError):
        GatedBlock(128, 3, 1, 256, None)
    with pytest.raises(ValueError):
        GatedBlock(128, 4, 3, 256, None)
    with pytest.raises(ValueError):
        GatedDecoder(vocab=8, d_model=16, layers=1, heads=2, kv_heads=1, hidden=8, checkpoint="int4")


@pytest.mark.gpu
def test_gpu_gradients_are_the_cpu_forms():
    torch.manual_seed(2)
    host = gated_tiny()
    device = gated_tiny()
    device.load_state_dict(host.state_dict())
    device = device.cuda()
    a, b = host(*_batch("cpu")), device(*_batch("cuda"))
    a.backward(), b.backward()
    assert abs(a.item() - b.item()) < 1e-4
    for (name, p), q in zip(host.named_parameters(), device.parameters()):
        # four layers in fp32, sums of at most some thousand terms each: far below a thousandth of the gradient's size
        assert (p.grad - q.grad.cpu()).norm() <= 1e-3 * p.grad.norm(), name


@pytest.mark.gpu
@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_a_ddp_step_under_autocast_runs_on_the_kernels(checkpoint):
    import torch.distributed as dist

    from mccl_b200.optim import FusedAdamW
    from mccl_b200.parallel import wrap_ddp
    native = mccl_b200.require_native()
    created = not dist.is_initialized()
    if created:
        dist.init_process_group("mccl", store=dist.HashStore(), rank=0, world_size=1)
    try:
        torch.manual_seed(0)
        model = wrap_ddp(gated_tiny(checkpoint=checkpoint).cuda(), device_ids=[0])
        opt = FusedAdamW(model.parameters(), lr=3e-3)
        x, y = _batch("cuda")
        losses = []
        for _ in range(12):
            opt.zero_grad()
            before = native._kernel_launches()
            with torch.autocast("cuda", dtype=torch.bfloat16):
                loss = model(x, y)
            loss.backward()
            # a layer's heads take three launches, its gated block four, packed rows three times two more
            assert native._kernel_launches() - before >= 4 * (13 if checkpoint else 7)
            opt.step()
            losses.append(loss.item())
        assert losses[-1] < losses[0] - 2
    finally:
        if created:
            dist.destroy_process_group()


def test_example_two_cpu_ranks(tmp_path):
    stats = tmp_path / "ddp.json"
    r = subprocess.run([sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node", "2", "--master-addr", "127.0.0.1",
                        "--master-port", "29877", "examples/ddp_dummy_train.py", "--cpu", "--model", "gated-tiny", "--checkpoint", "int8",
                        "--steps", "4", "--warmup", "1", "--batch-size", "2", "--save-stats", str(stats)],
                       cwd=ROOT, env=dict(os.environ), capture_output=True, text=True, timeout=240)
    assert r.returncode == 0, r.stderr[-2000:]
    s = json.loads(stats.read_text())
    assert s["world_size"] == 2 and len(s["step_times"]) == 4
