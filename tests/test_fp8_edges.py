"""Products in 8 bits and the layer made of them where their arithmetic and their sizes come to their ends."""
import pytest
import torch

import fp8_reference as ref
from torchmpi_b200._lib import lib
from torchmpi_b200.ops import fp8

gpu = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]
BF, HALF, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF, HALF, FP32])
@pytest.mark.parametrize("T,K,N", [(3, 64, 16), (32, 64, 40), (40, 64, 15), (40, 8192, 16), (300, 256, 523), (300, 64, 520)])
def test_gelu_of_infinities(T, K, N, dtype, device):
    """-inf times Phi(-inf) is no number, +inf stays: whatever kernel the number of tokens leads to, and beside finite columns that do not notice."""
    inf, nan = float("inf"), float("nan")
    lowest = torch.finfo(dtype).min
    b = torch.zeros(N)
    b[:8] = torch.tensor([-inf, lowest, inf, -1024.0, 2.0, nan, -inf, 0.0])
    b[-1] = -inf
    b = b.to(dtype).to(device)
    x, w = torch.zeros(T, K, dtype=dtype, device=device), torch.zeros(N, K, dtype=dtype, device=device)
    want = torch.where(torch.isnan(b) | (b == -inf), nan, torch.where(b < 0, 0, b).double() * ref.phi(b.double())).cpu().expand(T, -1)
    with torch.no_grad():
        results = [fp8.linear(x, w, b, gelu=True), fp8.linear(x, fp8.quantize(w), b, gelu=True)]
    results.append(fp8.linear(x.clone().requires_grad_(), w, b, gelu=True))
    for y in results:
        y = y.detach().double().cpu()
        assert torch.equal(torch.isnan(y), torch.isnan(want))
        assert torch.equal(torch.isinf(y), torch.isinf(want))
        fine = torch.isfinite(want)
        assert ((y - want)[fine].abs() <= (3e-6 + ref.half_step(want, dtype))[fine]).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T", [5, 200])
def test_gelu_of_sums_beyond_the_type(T, device):
    """Sums that bf16 and fp32 do not hold are infinities of either sign before the GELU."""
    x, w = torch.zeros(T, 128), torch.zeros(24, 128)
    x[1], x[2] = 2.0 ** 126, 2.0 ** 126
    w[3], w[4] = 2.0, -2.0
    y = fp8.linear(x.to(BF).to(device), w.to(BF).to(device), None, gelu=True).double().cpu()
    want = torch.zeros(T, 24).double()
    want[1:3, 3], want[1:3, 4] = float("inf"), float("nan")
    assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(y.nan_to_num(0), want.nan_to_num(0))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("gelu", [False, True])
@pytest.mark.parametrize("T,N", [(5, 0), (0, 0), (0, 3)])
def test_layers_without_outputs_or_tokens(T, N, gelu, device):
    """Nothing comes of them, and the gradients are zeros of the inputs' shapes."""
    x, w, b = (torch.randn(s, device=device).to(BF).requires_grad_() for s in ((T, 7), (N, 7), (N,)))
    y = fp8.linear(x, w, b, gelu)
    assert y.shape == (T, N) and y.dtype == BF
    for t, d in zip((x, w, b), torch.autograd.grad(y.sum(), (x, w, b))):
        assert d.shape == t.shape and d.dtype == t.dtype and not d.any()
    kept = fp8.quantize(w.detach())
    assert fp8.linear(x.detach(), kept, b.detach(), gelu).shape == (T, N) and fp8.matmul(fp8.quantize(x.detach()), kept).shape == (T, N)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF, HALF, FP32])
def test_the_slope_of_the_gelu(dtype, device):
    """For one token and a gradient of ones the bias' gradient is the slope itself.  Phi is within 7.5e-8 (half of erf's 1.5e-7), its fp32 polynomial within 1.5e-7, the exponential within 2^-22 of itself and the reciprocal
    within 2^-23: 6e-7 together, and the rounding."""
    z = torch.arange(-2 ** 15, 2 ** 15, dtype=torch.int32).to(torch.int16).view(BF).float() if dtype == BF else torch.linspace(-9, 9, 40001)
    z = z[z.abs() <= 9].to(dtype)
    x, w, b = torch.zeros(1, 16, dtype=dtype, device=device), torch.zeros(z.numel(), 16, dtype=dtype, device=device), z.to(device).requires_grad_()
    y = fp8.linear(x, w, b, gelu=True)
    slope, = torch.autograd.grad(y, b, torch.ones_like(y))
    want = ref.slope(z.double())
    ref.close(slope, want, 6e-7 + ref.half_step(want, dtype) * (1 + 2.0 ** -10), "slope")
