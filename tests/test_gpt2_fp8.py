"""GPT-2 with products in 8 bits, and trained with AdamW through the engine."""
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import fp8_reference as ref
from mp_util import run_ranks
from torchmpi_b200.engine import AllReduceSGDEngine
from torchmpi_b200.models import gpt2
from torchmpi_b200.ops import adamw, fp8

gpu = pytest.mark.gpu


def _net(device, **form):
    torch.manual_seed(3)
    net = gpt2.gpt2_tiny(n_head=2, n_embd=128, block_size=128, vocab_size=512, tc_linear=device == "cuda", fp8=True, **form).to(device)
    idx, target = torch.randint(0, 512, (2, 128), device=device), torch.randint(0, 512, (2, 128), device=device)
    return (net.to(torch.bfloat16) if device == "cuda" else net), idx, target


def _step(net, idx, target):
    loss = gpt2.LMLoss()(net(idx), target)
    return loss, torch.autograd.grad(loss, list(net.parameters()))


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("form", [dict(), dict(act8=True), dict(n_expert=4)], ids=str)
def test_trains(form, device):
    net, idx, target = _net(device, **form)
    before = fp8.launch_count
    loss, grads = _step(net, idx, target)
    # a layer: one launch of quantization and one product forward; one and two backward
    assert device == "cpu" or fp8.launch_count - before >= 2 * 5 * (2 if form else 4)
    assert torch.isfinite(loss) and all(g.isfinite().all() and g.any() for g in grads if not form)
    again = _step(net, idx, target)
    assert torch.equal(loss, again[0])
    if device == "cuda":
        fp8.check_status()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_a_blocks_layers_against_64_bits(device):
    """The layers inside a running model: inputs and gradients are taken there, results compared with the formulas."""
    net, idx, target = _net(device)
    held = {}
    for name in ("qkv", "proj", "out"):
        def look(module, args, out, name=name):
            held[name] = dict(x=args[0].detach(), y=out.detach())
            out.register_hook(lambda g: held[name].update(dy=g.detach()))
        getattr(net.blocks[1], name).register_forward_hook(look)
    gpt2.LMLoss()(net(idx), target).backward()
    for name, h in held.items():
        m = getattr(net.blocks[1], name)
        x, y, dy = (h[k].reshape(-1, h[k].shape[-1]).cpu() for k in ("x", "y", "dy"))
        w, b = m.weight.detach().cpu(), m.bias.detach().cpu()
        want, bound = ref.product(ref.kept(x), ref.kept(w), b)
        ref.close(y, want, bound + ref.half_step(want.abs() + bound, y.dtype), name)
        want, bound = ref.product(ref.kept(dy.t()), ref.kept(x.t()))
        ref.close(m.weight.grad, want, bound + ref.half_step(want.abs() + bound, y.dtype), name + ".weight")


@gpu
def test_generates_a_token_with_kept_weights():
    """The MLP of a block for one token, weights in 8 bits, as the layers themselves form it."""
    net, idx, target = _net("cuda")
    block, x = net.blocks[0], torch.randn(1, 1, 128, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        fc, out = fp8.quantize(block.fc.weight), fp8.quantize(block.out.weight)
        h = fp8.linear(x, fc, block.fc.bias, gelu=True)
        assert torch.equal(block.out(block.fc(x)), fp8.linear(h, out, block.out.bias))


# ---------------------------------------------------------------- the engine
def _mlp(bits):
    from torchmpi_b200.models.mlp import MLP
    torch.manual_seed(5)
    net = MLP()
    g = torch.Generator().manual_seed(6)
    data = [{"input": torch.rand(16, 1, 28, 28, generator=g), "target": torch.randint(0, 10, (16,), generator=g)} for _ in range(4)]
    return net, data, lambda params: adamw.AdamW(params, weight_decay=0.1, bits=bits, max_norm=0.5)


def _engine_step(rank, world, bits):
    import torchmpi_b200 as mpi
    from torchmpi_b200 import nn as mpinn
    mpi.start(with_cuda=False)
    net, data, make = _mlp(bits)
    engine = AllReduceSGDEngine(gradient_scale=1.0 / world, optimizer=make)
    engine.train(net, torch.nn.NLLLoss(), data, lr=0.01, maxepoch=1)
    mpinn.check_with_allreduce(net)
    assert int(engine.own_optimizer.state[next(net.parameters())]["step"]) == 4
    flat = torch.cat([p.detach().reshape(-1) for p in net.parameters()])
    mpi.stop()
    return flat.tolist()


@pytest.mark.parametrize("bits", [8, 32])
def test_the_engine_steps_with_an_optimizer(bits):
    """Two ranks with the same data: the mean of two equal gradients is that gradient, so the weights are those of a plain loop."""
    got = run_ranks(_engine_step, 2, bits, timeout=300)
    net, data, make = _mlp(bits)
    opt = make(list(net.parameters()))
    for s in data:
        opt.zero_grad()
        torch.nn.NLLLoss()(net(s["input"]), s["target"]).backward()
        opt.step(0.01)
    assert got[0] == got[1] == torch.cat([p.detach().reshape(-1) for p in net.parameters()]).tolist()


def test_the_engine_refuses_two_updates():
    for options in (dict(fused=True), dict(momentum=0.9), dict(weight_decay=0.1), dict(nesterov=True), dict(dampening=0.5)):
        with pytest.raises(ValueError):
            AllReduceSGDEngine(optimizer=lambda params: None, **options)


def _example(launcher, **env):
    examples = Path(__file__).resolve().parent.parent / "examples"
    return subprocess.run([sys.executable, *launcher, str(examples / "gpt2_dataparallel.py")], capture_output=True, text=True, timeout=600, cwd=str(examples),
                          env=dict(os.environ, EXAMPLE_FP8="1", PYTHONPATH=str(examples.parent), **env))


@pytest.mark.parametrize("bits", ["0", "8", "32"])
def test_two_ranks_train_it_data_parallel(bits):
    """The example over gloo: the replicas stay equal, which it checks itself."""
    r = _example(("-m", "torchmpi_b200.launch", "--nproc", "2"), EXAMPLE_ADAMW=bits, OMP_NUM_THREADS="2")
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-3000:]


@gpu
@pytest.mark.parametrize("bits", ["0", "8", "32"])
def test_the_example_runs_on_the_kernels(bits):
    r = _example((), EXAMPLE_ADAMW=bits, EXAMPLE_DEVICE="cuda")
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-3000:]
