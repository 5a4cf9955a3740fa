"""GPT-2 with layers of experts and with 8-bit checkpoints in its blocks."""
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import expert_reference as ref
from torchmpi_b200.models import gpt2
from torchmpi_b200.ops import act8, experts

gpu = pytest.mark.gpu
FORMS = [dict(n_expert=4), dict(n_expert=8, expert_k=3, act8=True), dict(act8=True)]


def _step(net, idx, target):
    loss = gpt2.LMLoss()(net(idx), target)
    return loss, torch.autograd.grad(loss, list(net.parameters()))


@pytest.mark.parametrize("form", FORMS, ids=str)
def test_trains_on_the_cpu(form):
    torch.manual_seed(0)
    net = gpt2.gpt2_tiny(n_head=2, n_embd=32, block_size=16, vocab_size=64, **form)
    idx, target = torch.randint(0, 64, (2, 16)), torch.randint(0, 64, (2, 16))
    loss, grads = _step(net, idx, target)
    assert torch.isfinite(loss) and all(g.isfinite().all() for g in grads)
    named = dict(zip((n for n, _ in net.named_parameters()), grads))
    for n in ("blocks.0.experts.gate.weight", "blocks.0.experts.w1", "blocks.1.experts.b2") if form.get("n_expert") else ("blocks.0.fc.weight", "blocks.1.out.bias"):
        assert named[n].any(), n


def test_eight_bits_change_little_and_hooks_are_called():
    """The forward pass is the same with 8-bit checkpoints; a hooked layer is called as a layer."""
    torch.manual_seed(1)
    a = gpt2.gpt2_tiny(n_head=2, n_embd=32, block_size=16, vocab_size=64)
    b = gpt2.gpt2_tiny(n_head=2, n_embd=32, block_size=16, vocab_size=64, act8=True)
    b.load_state_dict(a.state_dict())
    idx = torch.randint(0, 64, (2, 16))
    assert torch.allclose(a(idx), b(idx), atol=1e-5)
    seen = []
    b.blocks[0].fc.register_forward_hook(lambda m, i, o: seen.append(o.shape))
    b(idx)
    assert seen == [(2, 16, 128)]


def test_experts_see_every_token_alone():
    """With one expert and k = 1 the layer is an MLP with its weights."""
    torch.manual_seed(2)
    m = experts.Experts(16, 32, 1, 1)
    x = torch.randn(3, 5, 16)
    want = torch.nn.functional.gelu(x @ m.w1[0].t() + m.b1[0]) @ m.w2[0].t() + m.b2[0]
    assert torch.allclose(m(x), want, atol=1e-5)


@gpu
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_trains_on_the_kernels(form):
    torch.manual_seed(3)
    net = gpt2.gpt2_tiny(n_head=2, n_embd=128, block_size=128, vocab_size=512, tc_linear=True, **form).cuda().to(torch.bfloat16)
    idx, target = torch.randint(0, 512, (2, 128), device="cuda"), torch.randint(0, 512, (2, 128), device="cuda")
    before = experts.launch_count, act8.launch_count
    loss, grads = _step(net, idx, target)
    assert experts.launch_count > before[0] and (act8.launch_count > before[1] or not form.get("act8") or form.get("n_expert"))
    assert torch.isfinite(loss) and all(g.isfinite().all() for g in grads)
    again = _step(net, idx, target)
    assert torch.equal(loss, again[0])
    experts.check_status()


@gpu
def test_a_blocks_experts_against_64_bits():
    """The layer inside a running model: its inputs and its output's gradient are taken there, its results compared with the formulas."""
    torch.manual_seed(4)
    net = gpt2.gpt2_tiny(n_layer=1, n_head=2, n_embd=128, block_size=128, vocab_size=512, tc_linear=True, n_expert=8).cuda().to(torch.bfloat16)
    m = net.blocks[0].experts
    held = {}

    def look(module, args, out):
        held["x"], held["y"] = args[0].detach(), out.detach()
        out.register_hook(lambda g: held.setdefault("dy", g.detach()))
        args[0].register_hook(lambda g: held.setdefault("dx_and_gate", g.detach()))
    m.register_forward_hook(look)
    idx, target = torch.randint(0, 512, (2, 128), device="cuda"), torch.randint(0, 512, (2, 128), device="cuda")
    gpt2.LMLoss()(net(idx), target).backward()
    x, dy = held["x"].reshape(-1, 128), held["dy"].reshape(-1, 128)
    r = experts.route(torch.nn.functional.linear(x, m.gate.weight) if x.shape[0] % 8 else _gate(x, m), 2)
    y, dx, dwt, dw1, db1, dw2, db2 = ref.experts(x, r.weights, r.chosen, m.w1.detach(), m.b1.detach(), m.w2.detach(), m.b2.detach(), dy, False, exact_z=False)
    ref.close(held["y"].reshape(-1, 128), y, "y")
    for name, got, want in (("dw1", m.w1.grad, dw1), ("db1", m.b1.grad, db1), ("dw2", m.w2.grad, dw2), ("db2", m.b2.grad, db2)):
        ref.close(got, want, name)


def _gate(x, m):
    from torchmpi_b200.ops import gemm
    return gemm.linear(x, m.gate.weight).detach()


def _example(launcher, **env):
    examples = Path(__file__).resolve().parent.parent / "examples"
    return subprocess.run([sys.executable, *launcher, str(examples / "gpt2_dataparallel.py")], capture_output=True, text=True, timeout=600, cwd=str(examples),
                          env=dict(os.environ, EXAMPLE_EXPERTS="4", EXAMPLE_ACT8="1", PYTHONPATH=str(examples.parent), **env))


def test_two_ranks_train_it_data_parallel():
    """The example over gloo: the replicas stay equal, which it checks itself."""
    r = _example(("-m", "torchmpi_b200.launch", "--nproc", "2"))
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-3000:]


@gpu
def test_the_engine_trains_it():
    """The fused optimizer's flat buckets hold the experts' three-dimensional weights."""
    r = _example((), EXAMPLE_DEVICE="cuda")
    assert r.returncode == 0 and "accuracy" in r.stdout, r.stdout[-2000:] + r.stderr[-3000:]
