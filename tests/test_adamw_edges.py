"""AdamW where its arithmetic and its inputs come to their ends."""
import pytest
import torch

from torchmpi_b200.ops import adamw

gpu = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]
BF, HALF, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", [BF, FP32])
@pytest.mark.parametrize("lr,beta1", [(0.5, 0.9), (0.86, 0.9), (1.0, 0.9), (0.1, 0.99), (0.01, 0.999), (100.0, 0.9), (1e4, 0.999), (1e20, 0.0)])
def test_no_gradient_no_eps_at_any_rate(lr, beta1, dtype, bits, device):
    """Elements that never had a gradient stay, also with eps = 0 and whatever lr / (1 - beta1) is, which divides the least divisor."""
    p = torch.ones(200, device=device, dtype=dtype).requires_grad_(True)
    opt = adamw.AdamW([p], eps=0.0, bits=bits, weight_decay=0.0, lr=lr, betas=(beta1, 0.999))
    for _ in range(2):
        p.grad = torch.zeros_like(p)
        p.grad[3] = 2.0
        opt.step()
        rest = torch.cat([p.detach()[:3], p.detach()[4:]])
        assert (rest == 1).all()
        for flat in (*opt.moments(), opt.masters()):
            assert flat is None or (flat[200:] == 0).all()
    # equal gradients: each step has the rate's length.  The averages of 8 bits hold the block's largest element, itself, to 2^-20
    want = 1 - 2 * lr
    got = float((opt.state[p]["master"] if dtype != FP32 else p.detach())[3])
    assert abs(got - want) <= 2.0 ** -17 * (1 + 2 * lr)
