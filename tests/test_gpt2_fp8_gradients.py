"""The gradients of every form of GPT-2 with products in 8 bits."""
import pytest
import torch

from torchmpi_b200.models import gpt2
from torchmpi_b200.ops import fp8

gpu = pytest.mark.gpu


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("form", [dict(), dict(act8=True), dict(n_expert=4), dict(n_expert=4, act8=True)], ids=str)
def test_every_parameter_has_its_gradient(form, device):
    """Finite ones everywhere, none of nothing (experts alone may get no token), and the same bits again."""
    torch.manual_seed(3)
    net = gpt2.gpt2_tiny(n_head=2, n_embd=128, block_size=128, vocab_size=512, tc_linear=device == "cuda", fp8=True, **form).to(device)
    idx, target = torch.randint(0, 512, (2, 128), device=device), torch.randint(0, 512, (2, 128), device=device)
    net = net.to(torch.bfloat16) if device == "cuda" else net
    names, params = zip(*net.named_parameters())
    step = lambda: torch.autograd.grad(gpt2.LMLoss()(net(idx), target), params)      # noqa: E731
    grads, again = step(), step()
    last = f"blocks.{len(net.blocks) - 1}."
    compared = 0
    for name, g, h in zip(names, grads, again):
        assert g.isfinite().all(), name
        assert g.any() or ".experts." in name, name
        # on the GPU the gradient of attention's queries is summed in any order: what lies behind the last block's attention does not depend on it
        if device == "cpu" or (name.startswith(last) and not any(part in name for part in ("ln1", "qkv"))) or name.startswith("ln_f"):
            assert torch.equal(g, h), name
            compared += 1
    assert compared >= 6
    if form.get("n_expert"):
        assert any(g.any() for name, g in zip(names, grads) if ".experts." in name)
    if device == "cuda":
        fp8.check_status()
