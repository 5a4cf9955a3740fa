"""Layers of experts and 8-bit checkpoints on tensors of 64 bits: chosen, multiplied and added as those hold them."""
import math

import pytest
import torch

from torchmpi_b200.ops import act8, experts

gpu = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]
F64 = torch.float64


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("renormalize", [True, False])
def test_the_choice_among_logits_of_64_bits(renormalize, device):
    """Logits that differ by less than 32 bits hold, or beyond their range, are different."""
    l = torch.tensor([[1.0, 1.0 + 2.0 ** -40, 1.0 - 2.0 ** -40, 0.0], [1e300, 2e300, -1e300, 0.0], [-1e300, -math.inf, -2e300, -math.inf]], dtype=F64, device=device)
    r = experts.route(l, 2, renormalize)
    assert r.chosen.tolist() == [[1, 0], [1, 0], [0, 2]] and r.offsets[-1] == 6
    assert r.weights.dtype == torch.float32
    p = torch.softmax(torch.gather(l, 1, r.chosen.long()) if renormalize else l, 1)
    want = p if renormalize else torch.gather(p, 1, r.chosen.long())
    assert bool(((r.weights.double() - want).abs() <= (2.0 ** -24 + 2.0 ** -48) * want).all())      # one rounding to fp32, of what 64 bits are good for
    leaf = l[:1].clone().requires_grad_(True)
    dw = torch.tensor([[1.0, -2.0]], device=device)
    (got,) = torch.autograd.grad(experts.route(leaf, 2, renormalize).weights, leaf, dw)
    other = l[:1].clone().requires_grad_(True)
    p = torch.softmax(other[:, [1, 0]], 1) if renormalize else torch.softmax(other, 1)[:, [1, 0]]
    (want,) = torch.autograd.grad(p, other, dw.double())
    assert got.dtype == F64 and bool(((got - want).abs() <= 16 * 2.0 ** -53 * 3).all())      # some roundings of terms that add up to 3 at most
