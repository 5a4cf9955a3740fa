"""Every form of the products in 8 bits inside the layer, against 64 bits: tiles of 128, 192 and 256 columns with several tiles to a CTA pair, slices of K, each with the bias sums, the GELU
and the pre-activation."""
import ctypes

import pytest
import torch

import fp8_reference as ref
from torchmpi_b200._lib import lib
from torchmpi_b200.ops import fp8

gpu = pytest.mark.gpu
BF, HALF, FP32 = torch.bfloat16, torch.float16, torch.float32

# T, K, N, and the forms (columns of a tile, whether K is cut) of the forward product, the input gradient and the weights' gradient on 74 pairs of SMs
FORMS = [
    ((4096, 128, 136), (128, False), (128, False), (128, True)),           # bias sums beside slices
    ((300, 8192, 523), (192, True), (256, False), (192, False)),           # a GELU behind slices, odd rows
    ((300, 8192, 64), (128, True), (256, False), (128, False)),
    ((6144, 128, 2048), (256, False), (128, False), (128, True)),          # two and three tiles to a pair, whose accumulators overlap
    ((2304, 64, 4096), (256, False), (128, True), (128, False)),
    ((2560, 64, 5760), (192, False), (128, True), (128, False)),           # four and five
    ((4500, 64, 4100), (192, False), (128, True), (128, True)),            # rows that the TMA unit does not store
    ((3500, 64, 3500), (256, False), (128, True), (128, True)),
]


def _form(M, N, K):
    columns, slices = ctypes.c_int(), ctypes.c_int()
    assert lib.tmpi_fp8_product_form(M, N, K, columns, slices) == 0
    assert (slices.value > 1) == (lib.tmpi_fp8_product_workspace_bytes(M, N, K) > 0)
    return columns.value, slices.value > 1


def test_refuses_sizes_that_are_none():
    columns, slices = ctypes.c_int(), ctypes.c_int()
    for sizes in ((0, 4, 8), (4, 0, 8), (4, 4, 0), (2 ** 30 + 1, 4, 8)):
        assert lib.tmpi_fp8_product_form(*sizes, columns, slices) != 0


@gpu
@pytest.mark.parametrize("case", FORMS, ids=lambda c: "x".join(map(str, c[0])))
def test_the_cases_are_of_their_forms(case):
    (T, K, N), forward, dx, dw = case
    assert (_form(T, N, K), _form(T, K, N), _form(N, K, T)) == (forward, dx, dw)


@gpu
@pytest.mark.parametrize("dtype", [BF, HALF, FP32])
@pytest.mark.parametrize("gelu", [False, True])
@pytest.mark.parametrize("T,K,N", [c[0] for c in FORMS], ids=str)
def test_layer(T, K, N, gelu, dtype):
    """Inputs whose sums fp32 holds exactly, so that the pre-activation is one number on both sides; the slope and the GELU are within 3e-6 of the exact ones, and where that moves a rounding, or
    its 8 bits, the bound takes in both."""
    g = torch.Generator().manual_seed(T + K + N)
    x, w, b = ref.grid(g, (T, K), 1 / 4, 2).cuda(), ref.grid(g, (N, K), 1 / 32, 1 / 4).cuda(), ref.grid(g, (N,), 1 / 16, 1).cuda()
    dy = torch.randn(T, N, generator=g).to(dtype).cuda()
    z = (x @ w.t() + b).to(dtype).double()
    leaves = [t.to(dtype).requires_grad_(True) for t in (x, w, b)]
    assert all(torch.equal(leaf.detach().double(), t) for leaf, t in zip(leaves, (x, w, b)))
    y = fp8.linear(*leaves, gelu=gelu)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    want = z * ref.phi(z) if gelu else z
    ref.close(y, want.cpu(), (ref.half_step(want, dtype) + 3e-6 + 2.0 ** -22 * want.abs() if gelu else torch.zeros_like(want)).cpu(), "y")
    dz, slack = dy.double(), torch.zeros_like(want)
    if gelu:
        dz = dy.double() * ref.slope(z)
        slack = 3e-6 * dy.double().abs() + 2.0 ** -22 * dz.abs()
    near = [(dz + s * slack).to(dtype).double() for s in ((-1, 0, 1) if gelu else (0,))]

    def spread(f):
        forms = [f(t) for t in near]
        least, most = forms[0], forms[0]
        for t in forms[1:]:
            least, most = torch.minimum(least, t), torch.maximum(most, t)
        return forms[len(forms) // 2], most - least
    for name, got, (q, off), other in (("dx", dx, spread(ref.kept), w.t()), ("dw", dw, spread(lambda t: ref.kept(t.t())), x.t())):
        want, bound = ref.product(q, other)
        bound = bound + off @ other.abs().t()
        ref.close(got, want.cpu(), (bound + ref.half_step(want.abs() + bound, dtype)).cpu(), name)
    rounded, off = spread(lambda t: t)
    want, bound = rounded.sum(0), off.sum(0) + T * 2.0 ** -24 * rounded.abs().sum(0)
    ref.close(db, want.cpu(), (bound + ref.half_step(want.abs() + bound, dtype)).cpu(), "db")
    again = torch.autograd.grad(fp8.linear(*leaves, gelu=gelu), leaves, dy)
    assert all(torch.equal(p, q) for p, q in zip(again, (dx, dw, db)))
    with torch.no_grad():                              # the GELU alone, without what a backward pass keeps
        for weight in (leaves[1], fp8.quantize(leaves[1])):
            assert torch.equal(fp8.linear(leaves[0], weight, leaves[2], gelu), y)
    fp8.check_status()
