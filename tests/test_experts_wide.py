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


def _f64(device, *sizes, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(s, generator=g, dtype=F64).to(device).requires_grad_(True) for s in sizes]


def _near(got, want):
    """64 bits: sums of up to 40 terms of a few units"""
    assert got.dtype == F64 and bool(((got - want).abs() <= 1e-13 * (1 + want.abs())).all()), float((got - want).abs().max())


@pytest.mark.parametrize("device", DEVICES)
def test_products_and_rows_of_64_bits(device):
    x, w, b = _f64(device, (7, 5), (3, 6, 5), (3, 6))
    off = torch.tensor([0, 3, 3, 6], dtype=torch.int32, device=device)
    for gelu in (False, True):
        f = torch.nn.functional.gelu if gelu else (lambda z: z)
        y = experts.grouped_linear(x, w, b, off, gelu)
        want = torch.cat([f(x[:3] @ w[0].t() + b[0]), f(x[3:6] @ w[2].t() + b[2]), torch.zeros(1, 6, dtype=F64, device=device)])
        _near(y, want)
        dy = torch.randn(7, 6, dtype=F64, generator=torch.Generator().manual_seed(1)).to(device)
        for a, c in zip(torch.autograd.grad(y, (x, w, b), dy), torch.autograd.grad(want, (x, w, b), dy)):
            _near(a, c)
    r = experts.route(torch.tensor([[1.0, 2.0, 0.0], [0.0, -math.inf, 1.0], [-math.inf] * 3], device=device), 2)
    rows, = _f64(device, (6, 5), seed=2)
    _near(experts.combine(rows, r), (rows[r.place.long().clamp_min(0)] * torch.where(r.place >= 0, r.weights, 0).double().unsqueeze(2)).sum(1))
    _near(experts.dispatch(x[:3], r)[:4], x[:3][r.order[:4].long() // 2])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kept8", [False, True])
def test_a_layer_of_64_bits(kept8, device):
    """What is kept in 8 bits is rounded there, and nothing else anywhere: inputs and pre-activations of few bits give the gradients of the formula."""
    g = torch.Generator().manual_seed(3)
    few = lambda *s: torch.randint(-2, 3, s, generator=g).double().to(device).requires_grad_(True)
    x, w1, b1 = few(6, 4), few(3, 8, 4), few(3, 8)
    with torch.no_grad():
        w1.clamp_(-1, 1)                                        # |x w1^T + b1| <= 10: e4m3 holds the integers up to 16
    w2, b2 = _f64(device, (3, 4, 8), (3, 4))
    dy = torch.randn(6, 4, dtype=F64, generator=g).to(device)
    r = experts.route(torch.randn(6, 3, generator=g).to(device), 2)
    weights = r.weights.clone().requires_grad_(True)
    leaves = (x, weights, w1, b1, w2, b2)
    y = experts.mlp(x, r._replace(weights=weights), w1, b1, w2, b2, act8=kept8)
    want = 0
    for j in range(2):
        e = r.chosen[:, j].long()
        z = torch.einsum("tc,thc->th", x, w1[e]) + b1[e]
        want = want + weights[:, j:j + 1] * (torch.einsum("th,tch->tc", torch.nn.functional.gelu(z), w2[e]) + b2[e])
    _near(y, want)
    for a, c in zip(torch.autograd.grad(y, leaves, dy), torch.autograd.grad(want, leaves, dy)):
        if a.dtype == F64:
            _near(a, c)
        else:                                                   # the weights are fp32, and so is their gradient
            assert bool(((a - c).abs() <= 2.0 ** -23 * (1 + c.abs())).all())


@pytest.mark.parametrize("device", DEVICES)
def test_an_mlp_of_64_bits_with_8_bit_checkpoints(device):
    g = torch.Generator().manual_seed(4)
    few = lambda *s: torch.randint(-1, 2, s, generator=g).double().to(device).requires_grad_(True)
    x, w1, b1 = few(6, 4), few(8, 4), few(8)
    w2, b2 = _f64(device, (5, 8), (5,))
    dy = torch.randn(6, 5, dtype=F64, generator=g).to(device)
    leaves = (x, w1, b1, w2, b2)
    y, want = act8.mlp(*leaves), torch.nn.functional.linear(torch.nn.functional.gelu(x @ w1.t() + b1), w2, b2)
    _near(y, want)
    for a, c in zip(torch.autograd.grad(y, leaves, dy), torch.autograd.grad(want, leaves, dy)):
        _near(a, c)
    z = torch.randint(-8, 9, (6, 5), generator=g).double().to(device).requires_grad_(True)
    value = torch.nn.functional.gelu(z)
    dz, h = act8.gelu_gradient(dy, act8.quantize(z))
    _near(h, value)
    _near(dz, torch.autograd.grad(value, z, dy)[0])
