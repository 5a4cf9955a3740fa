"""Matrices in 8 bits with a scale for each block of 128, their products and the linear layer made of them, against 64 bits."""
import os
import subprocess
import sys

import pytest
import torch
import torch.autograd.forward_ad as fwd
import torch.nn.functional as F

import fp8_reference as ref
from torchmpi_b200 import _native
from torchmpi_b200._lib import lib
from torchmpi_b200.ops import fp8

gpu = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]
BF, HALF, FP32 = torch.bfloat16, torch.float16, torch.float32


def _values(g, rows, cols, dtype, wild=True):
    """Rows of all sizes, blocks of zeros, numbers at the borders of the format, infinities and NaN."""
    x = torch.randn(rows, cols, generator=g) * torch.exp2(torch.randint(-12, 12, (rows, 1), generator=g).float())
    if wild:
        x[0, : min(cols, 3)] = 0
        x[-1, :128] = 0
        if cols > 130:
            x[rows // 2, 128] = float("inf")
            x[rows // 2, 130] = float("nan")
            x[rows // 3, :4] = torch.tensor([448.0, 449.0, 464.0, 1.0])
            x[rows // 4, :4] = torch.tensor([2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10, 448.0])
    return x.to(dtype)


def _same(got, want):
    """Bit for bit, whatever NaN's sign is."""
    q, p = got.q.cpu().view(torch.uint8), want.q.cpu().view(torch.uint8)
    assert q.shape == p.shape and got.cols == want.cols
    nan = (p & 127) == 127
    assert torch.equal((q & 127) == 127, nan) and torch.equal(q[~nan], p[~nan])
    host = lambda m: fp8.Block8(m.q.cpu(), m.scale.cpu(), m.cols)      # noqa: E731
    assert torch.equal(fp8.scales(host(got)), fp8.scales(host(want)))


SHAPES = [(1, 1), (3, 7), (1, 128), (5, 129), (128, 128), (130, 515), (127, 640), (257, 1000), (300, 24)]


# ---------------------------------------------------------------- the matrices
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF, HALF, FP32])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_matrices_are_the_definition(rows, cols, dtype, device):
    x = _values(torch.Generator().manual_seed(rows + cols), rows, cols, dtype)
    held = x.to(device)
    before = fp8.launch_count
    both = fp8.quantize_both(held)
    for m, t in ((fp8.quantize(held), x), (fp8.quantize_columns(held), x.t()), (both[0], x), (both[1], x.t())):
        assert m.q.shape == (t.shape[0], -(-t.shape[1] // 128) * 128) and m.cols == t.shape[1]
        want = ref.kept(t)
        got = fp8.dequantize(m, FP32).double().cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(0), want.nan_to_num(0))
        assert not m.q[:, t.shape[1]:].view(torch.uint8).any()                  # zeros behind the last column
        _same(m, fp8._quantize(t))
    assert device == "cpu" or fp8.launch_count == before + 7


@pytest.mark.parametrize("device", DEVICES)
def test_read_back_in_each_type(device):
    x = _values(torch.Generator().manual_seed(5), 77, 301, FP32, wild=False)
    m = fp8.quantize(x.to(device))
    for dtype in (BF, HALF, FP32, torch.float64):
        assert torch.equal(fp8.dequantize(m, dtype).cpu(), ref.kept(x).to(dtype))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows,cols", [(5, 1), (1, 3), (40, 5), (9, 7), (33, 9), (20, 127), (21, 129), (3, 255), (130, 257), (700, 1001)])
def test_read_back_over_the_ends_of_rows(rows, cols, device):
    """Rows that are no multiple of 16 bytes: pieces of the result go on over their ends and over those of blocks."""
    x = _values(torch.Generator().manual_seed(cols), rows, cols, FP32, wild=False)
    m = fp8.quantize(x.to(device))
    for dtype in (BF, HALF, FP32):
        assert torch.equal(fp8.dequantize(m, dtype).cpu(), ref.kept(x).to(dtype))


@gpu
@pytest.mark.parametrize("dtype", [BF, HALF, FP32])
def test_elements_from_any_address(dtype):
    buf = _values(torch.Generator().manual_seed(3), 1, 40 * 301 + 16, dtype).cuda().view(-1)
    for first in range(9):
        for cols, ld in ((301, 301), (128, 301), (136, 136), (5, 8), (264, 299)):
            x = buf[first:].as_strided((40, cols), (ld, 1))
            _same(fp8.quantize(x), fp8._quantize(x.cpu()))
            a, b = fp8.quantize_both(x)
            _same(a, fp8._quantize(x.cpu()))
            _same(b, fp8._quantize(x.cpu().t()))


def test_scales_are_where_the_documentation_says():
    x = torch.exp2(torch.randint(-9, 9, (300, 5), generator=torch.Generator().manual_seed(1)).float()).repeat_interleave(128, 1)
    m = fp8.quantize(x)
    s, at = fp8.scales(m), m.scale
    assert s.shape == (300, 5)
    for r in (0, 1, 31, 32, 127, 128, 200, 299):
        for b in range(5):
            assert at[((r // 128) * 2 + b // 4) * 512 + (r % 32) * 16 + r % 128 // 32 * 4 + b % 4] == s[r, b] == 127 + int(torch.log2(x[r, 128 * b])) - 8


@gpu
def test_views_rows_apart_and_odd_addresses():
    g = torch.Generator().manual_seed(2)
    wide = _values(g, 150, 700, BF).cuda()
    for x in (wide[:, 64:400], wide[:, 3:400], wide[3:, :640], wide.t(), wide.view(15, 10, 700), wide[::2], wide[:, :1], wide[5:6, 1:300]):
        flat = x.reshape(-1, x.shape[-1])
        _same(fp8.quantize(x), fp8._quantize(flat.cpu()))
        a, b = fp8.quantize_both(x)
        _same(a, fp8._quantize(flat.cpu()))
        _same(b, fp8._quantize(flat.cpu().t()))
    assert fp8.quantize(torch.zeros(4, 3, device="cuda", dtype=BF).expand(4, 3)).q.shape == (4, 128)


# ---------------------------------------------------------------- products
def _matrices(g, M, N, K, device):
    a, b = (torch.randn(n, K, generator=g) * torch.exp2(torch.randint(-4, 4, (n, 1), generator=g).float()) for n in (M, N))
    return fp8.quantize(a.to(device)), fp8.quantize(b.to(device)), ref.kept(a), ref.kept(b)


# tiles of 256, 192 and 128 columns, slices of K, rows that are no 16-byte multiples, ends inside tiles and groups of blocks
PRODUCTS = [(1, 1, 1), (40, 24, 128), (129, 257, 130), (256, 256, 1024), (300, 523, 640), (256, 192, 2048), (70, 8, 4096), (1000, 1016, 384), (2500, 2304, 520), (130, 4096, 264), (2300, 4001, 300)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF, HALF, FP32])
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_products(M, N, K, dtype, device):
    if device == "cpu" and M * N * K > 1 << 27:
        pytest.skip("the same operations as for the small ones")
    g = torch.Generator().manual_seed(M + N + K)
    a, b, av, bv = _matrices(g, M, N, K, device)
    bias = torch.randn(N, generator=g).to(dtype)
    for c in (None, bias):
        got = fp8.matmul(a, b, None if c is None else c.to(device), dtype)
        want, bound = ref.product(av, bv, c)
        assert got.dtype == dtype
        ref.close(got, want, bound + ref.half_step(want.abs() + bound, dtype), (M, N, K))
        assert torch.equal(got, fp8.matmul(a, b, None if c is None else c.to(device), dtype))
    if device == "cuda":
        fp8.check_status()


@gpu
def test_the_forms_of_the_products_are_met():
    """The sizes above take slices of K and whole sums."""
    assert {bool(lib.tmpi_fp8_product_workspace_bytes(*s)) for s in PRODUCTS} == {True, False}


@gpu
@pytest.mark.parametrize("dtype", [BF, HALF, FP32])
@pytest.mark.parametrize("T", [1, 8, 9, 16, 17, 32])
@pytest.mark.parametrize("K,N", [(4096, 1000), (8192, 24), (2100, 590), (3000, 2368), (127, 5000)])
def test_few_tokens(T, K, N, dtype):
    """One block, or two or four of them, to the blocks of K; odd numbers of weight rows."""
    g = torch.Generator().manual_seed(T + K + N)
    x, w, b = torch.randn(T, K, generator=g).to(dtype), (torch.randn(N, K, generator=g) * K ** -0.5).to(dtype), torch.randn(N, generator=g).to(dtype)
    for bias in (None, b):
        y = fp8.linear(x.cuda(), fp8.quantize(w.cuda()), None if bias is None else bias.cuda())
        want, bound = ref.product(ref.kept(x), ref.kept(w), bias)
        ref.close(y, want, bound + ref.half_step(want.abs() + bound, dtype), "y")
        assert torch.equal(y, fp8.linear(x.cuda(), fp8.quantize(w.cuda()), None if bias is None else bias.cuda()))
        one = fp8.linear(x[-1:].cuda(), fp8.quantize(w.cuda()), None if bias is None else bias.cuda())
        assert torch.equal(one[0], y[-1])                    # a token's results do not depend on the others


@gpu
def test_rows_and_columns_are_independent():
    """A row's results do not depend on the others, and NaN stays with its row or column."""
    g = torch.Generator().manual_seed(3)
    x, w = torch.randn(300, 512, generator=g).cuda(), torch.randn(270, 512, generator=g).cuda()
    clean = fp8.matmul(fp8.quantize(x), fp8.quantize(w), dtype=FP32)
    x[17, 200], w[33, 5] = float("nan"), float("inf")
    got = fp8.matmul(fp8.quantize(x), fp8.quantize(w), dtype=FP32)
    bad = torch.zeros_like(clean, dtype=torch.bool)
    bad[17], bad[:, 33] = True, True
    assert torch.equal(torch.isnan(got), bad) and torch.equal(got[~bad], clean[~bad])


# ---------------------------------------------------------------- the layer
def _layer(x, w, b, dy, gelu, device, needs=(True, True, True)):
    leaves = [None if t is None else t.to(device).requires_grad_(n) for t, n in zip((x, w, b), needs)]
    y = fp8.linear(*leaves, gelu=gelu)
    wanted = [t for t, n in zip(leaves, needs) if t is not None and n]
    got = iter(torch.autograd.grad(y, wanted, dy.to(device)))
    return y.detach(), [next(got) if t is not None and n else None for t, n in zip(leaves, needs)]


# T, K, N: single tokens, one of everything, odd widths, several tiles, slices of K in the weights' gradient
LAYERS = [(1, 128, 16), (1, 1, 1), (7, 130, 33), (32, 256, 128), (33, 64, 300), (200, 384, 136), (300, 1000, 523), (1030, 256, 264)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF, HALF, FP32])
@pytest.mark.parametrize("T,K,N", LAYERS)
def test_layer_without_gelu(T, K, N, dtype, device):
    g = torch.Generator().manual_seed(T + K + N)
    x = (torch.randn(T, K, generator=g) * torch.exp2(torch.randint(-3, 3, (T, 1), generator=g).float())).to(dtype)
    w, b, dy = (torch.randn(N, K, generator=g) * K ** -0.5).to(dtype), torch.randn(N, generator=g).to(dtype), torch.randn(T, N, generator=g).to(dtype)
    for bias in (b, None):
        y, (dx, dw, db) = _layer(x, w, bias, dy, False, device)
        pairs = [("y", y, ref.product(ref.kept(x), ref.kept(w), bias)), ("dx", dx, ref.product(ref.kept(dy), ref.kept(w.t()))), ("dw", dw, ref.product(ref.kept(dy.t()), ref.kept(x.t())))]
        if bias is not None:
            pairs.append(("db", db, (dy.double().sum(0), T * 2.0 ** -24 * dy.double().abs().sum(0))))
        for name, got, (want, bound) in pairs:
            assert got.dtype == dtype
            ref.close(got, want, bound + ref.half_step(want.abs() + bound, dtype), name)
        with torch.no_grad():                                  # few tokens take another kernel, whose sums are ordered otherwise
            again = fp8.linear(x.to(device), w.to(device), None if bias is None else bias.to(device))
            kept = fp8.linear(x.to(device), fp8.quantize(w.to(device)), None if bias is None else bias.to(device))
        want, bound = ref.product(ref.kept(x), ref.kept(w), bias)
        ref.close(again, want, bound + ref.half_step(want.abs() + bound, dtype), "without gradients")
        assert torch.equal(again, kept)
        assert all(torch.equal(p, q) for p, q in zip(_layer(x, w, bias, dy, False, device)[1], (dx, dw, db)) if q is not None)
    if device == "cuda":
        fp8.check_status()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF, HALF, FP32])
@pytest.mark.parametrize("T,K,N", LAYERS)
def test_layer_with_gelu(T, K, N, dtype, device):
    """Inputs whose sums fp32 holds exactly, so that the pre-activation is the same number on both sides.  The slope is within 2e-6 of the exact one: where that moves
    the gradient's rounding, or its 8 bits, the bound takes in both."""
    g = torch.Generator().manual_seed(T + K + N + 1)
    x, w, b = ref.grid(g, (T, K), 1 / 4, 2).to(dtype), ref.grid(g, (N, K), 1 / 32, 1 / 4).to(dtype), ref.grid(g, (N,), 1 / 16, 1).to(dtype)
    dy = torch.randn(T, N, generator=g).to(dtype)
    assert torch.equal(ref.kept(x), x.double()) and torch.equal(ref.kept(w.t()), w.t().double())
    z = (x.double() @ w.double().t() + b.double()).to(dtype).double()
    y, (dx, dw, db) = _layer(x, w, b, dy, True, device)
    want = z * ref.phi(z)
    ref.close(y, want, 3e-6 + 2.0 ** -22 * want.abs() + ref.half_step(want, dtype), "y")
    dz, slack = dy.double() * ref.slope(z), 2e-6 * dy.double().abs() + 2.0 ** -22 * (dy.double() * ref.slope(z)).abs()
    near = [(dz + s * slack).to(dtype).double() for s in (-1, 0, 1)]

    def spread(f):
        forms = torch.stack([f(t) for t in near])
        return forms[1], forms.amax(0) - forms.amin(0)
    rows, rows_off = spread(ref.kept)
    cols, cols_off = spread(lambda t: ref.kept(t.t()))
    for name, got, (q, off), other in (("dx", dx, (rows, rows_off), ref.kept(w.t())), ("dw", dw, (cols, cols_off), ref.kept(x.t()))):
        want, bound = ref.product(q, other)
        bound = bound + off @ other.abs().t()
        ref.close(got, want, bound + ref.half_step(want.abs() + bound, dtype), name)
    rounded, off = spread(lambda t: t)
    want, bound = rounded.sum(0), off.sum(0) + T * 2.0 ** -24 * rounded.abs().sum(0)
    ref.close(db, want, bound + ref.half_step(want.abs() + bound, dtype), "db")
    with torch.no_grad():
        kept = fp8.linear(x.to(device), fp8.quantize(w.to(device)), b.to(device), gelu=True)
    assert torch.equal(kept, fp8.linear(x.to(device), w.to(device), b.to(device), gelu=True).detach()) or T <= lib.tmpi_fp8_few_tokens()
    want = z * ref.phi(z)
    ref.close(kept, want, 3e-6 + 2.0 ** -22 * want.abs() + ref.half_step(want, dtype), "kept")
    if device == "cuda":
        fp8.check_status()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF, FP32])
@pytest.mark.parametrize("T", [3, 40])
def test_gelu_of_any_magnitude(T, dtype, device):
    """Far from zero nothing, or z itself, is left; NaN stays."""
    b = torch.tensor([-3e38, -1e30, -1e20, -1e12, -5000.0, -1000.0, -60.0, -9.0, 0.0, 9.0, 60.0, 1e12, 3e38, float("inf"), float("nan")]).to(dtype)
    x, w = torch.zeros(T, 64, dtype=dtype, device=device), torch.zeros(b.numel(), 64, dtype=dtype, device=device)
    want = torch.where(b < 0, 0, b).double().expand(T, -1)
    for weight in (w, fp8.quantize(w)):
        with torch.no_grad():
            y = fp8.linear(x, weight, b.to(device), gelu=True).double().cpu()
        assert torch.isnan(y[:, -1]).all() and torch.equal(y[:, 9:-1], want[:, 9:-1]) and (y[:, :9].abs() <= 3e-6).all(), y[0]
    y = fp8.linear(x.requires_grad_(), w, b.to(device), gelu=True).detach().double().cpu()
    assert torch.isnan(y[:, -1]).all() and torch.equal(y[:, 9:-1], want[:, 9:-1]) and (y[:, :9].abs() <= 3e-6).all(), y[0]


@pytest.mark.parametrize("device", DEVICES)
def test_gradients_against_differences(device):
    """With inputs that 8 bits hold the layer is an ordinary one: its gradients are the differences of a function of 64 bits."""
    g = torch.Generator().manual_seed(4)
    x, w, dy = ref.grid(g, (40, 256), 1 / 4, 2), ref.grid(g, (24, 256), 1 / 16, 1 / 2), ref.grid(g, (40, 24), 1 / 2, 2)
    b = ref.grid(g, (24,), 1 / 4, 1)
    _, grads = _layer(x.to(FP32), w.to(FP32), b.to(FP32), dy.to(FP32), False, device)
    f = lambda x, w, b: float((F.linear(x, w, b) * dy).sum())      # noqa: E731
    for at, grad in enumerate(grads):
        for _ in range(12):
            leaves = [x.clone(), w.clone(), b.clone()]
            i = int(torch.randint(0, leaves[at].numel(), (1,), generator=g))
            leaves[at].view(-1)[i] += 0.5
            up = f(*leaves)
            leaves[at].view(-1)[i] -= 1.0
            assert float(grad.reshape(-1)[i]) == up - f(*leaves)          # linear: the difference is exact


@gpu
def test_only_what_is_wanted():
    g = torch.Generator().manual_seed(6)
    x, w, b, dy = (torch.randn(s, generator=g).to(BF) for s in ((150, 200), (96, 200), (96,), (150, 96)))
    for gelu in (False, True):
        _, want = _layer(x, w, b, dy, gelu, "cuda")
        for needs in ((True, False, False), (False, True, False), (False, False, True), (True, True, False), (False, True, True), (True, False, True)):
            for got, full, n in zip(_layer(x, w, b, dy, gelu, "cuda", needs)[1], want, needs):
                assert not n or torch.equal(got, full)
        for needs in ((True, False, False), (False, True, False)):
            full = _layer(x, w, None, dy, gelu, "cuda")[1]
            for got, f, n in zip(_layer(x, w, None, dy, gelu, "cuda", needs)[1], full, needs):
                assert not n or torch.equal(got, f)
    leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
    y = fp8.linear(*leaves)
    assert torch.equal(torch.autograd.grad(y, leaves[1], dy.cuda())[0], _layer(x, w, b, dy, False, "cuda")[1][1])


@pytest.mark.parametrize("device", DEVICES)
def test_batches_expanded_inputs_and_gradients(device):
    g = torch.Generator().manual_seed(7)
    x, w = torch.randn(1, 6, 64, generator=g).to(BF).to(device).requires_grad_(), torch.randn(40, 64, generator=g).to(BF).to(device).requires_grad_()
    one = torch.randn(1, generator=g).to(BF).to(device).requires_grad_()
    y = fp8.linear(x.expand(3, 6, 64), w, one.expand(40))
    assert y.shape == (3, 6, 40)
    got = torch.autograd.grad(y.sum(), (x, w, one))                          # the incoming gradient is one number, expanded
    flat = x.detach().expand(3, 6, 64).reshape(18, 64).requires_grad_()
    bias = one.detach().expand(40).contiguous().requires_grad_()
    want = torch.autograd.grad(fp8.linear(flat, w, bias), (flat, w, bias), torch.ones(18, 40, device=device, dtype=BF))
    assert torch.equal(got[1], want[1])
    ref.close(got[0], want[0].double().cpu().view(3, 6, 64).sum(0, keepdim=True), ref.half_step(3 * want[0].double().cpu().view(3, 6, 64).abs().sum(0, keepdim=True), BF), "dx")
    assert float(got[2]) == 720.0                                            # 18 tokens, 40 outputs
    wide = torch.randn(50, 200, generator=g).to(BF).to(device)
    assert torch.equal(fp8.linear(wide[:, 8:72], w), fp8.linear(wide[:, 8:72].contiguous(), w))
    assert torch.equal(fp8.linear(wide[:, 5:69], w.detach().t().contiguous().t()), fp8.linear(wide[:, 5:69].contiguous(), w))


@pytest.mark.parametrize("device", DEVICES)
def test_no_tokens(device):
    x, w, b = (torch.zeros(s, device=device, dtype=BF, requires_grad=True) for s in ((2, 0, 64), (40, 64), (40,)))
    for gelu in (False, True):
        y = fp8.linear(x, w, b, gelu)
        assert y.shape == (2, 0, 40)
        for t, d in zip((x, w, b), torch.autograd.grad(y.sum(), (x, w, b))):
            assert d.shape == t.shape and not d.any()
    assert fp8.linear(x.detach(), fp8.quantize(w.detach()), b.detach()).shape == (2, 0, 40)
    assert fp8.dequantize(fp8.quantize(torch.zeros(0, 64, device=device))).shape == (0, 64)


@pytest.mark.parametrize("device", DEVICES)
def test_saved_tensors_on_the_host(device):
    g = torch.Generator().manual_seed(8)
    leaves = [torch.randn(s, generator=g).to(BF).to(device).requires_grad_() for s in ((70, 96), (80, 96), (80,))]
    dy = torch.randn(70, 80, generator=g).to(BF).to(device)
    want = torch.autograd.grad(fp8.linear(*leaves, gelu=True), leaves, dy)
    with torch.autograd.graph.save_on_cpu():
        y = fp8.linear(*leaves, gelu=True)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, dy), want))


def test_64_bits_on_operations():
    g = torch.Generator().manual_seed(9)
    x, w, dy = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((20, 200), (30, 200), (20, 30)))
    y, (dx, dw, _) = _layer(x, w, None, dy, False, "cpu")
    assert y.dtype == torch.float64
    for got, (a, b) in ((y, (x, w)), (dx, (dy, w.t())), (dw, (dy.t(), x.t()))):
        want = ref.kept(a.float()) @ ref.kept(b.float()).t()
        assert torch.allclose(got, want, rtol=1e-12, atol=1e-12)


# ---------------------------------------------------------------- refusals
@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    x, w, b = (torch.zeros(s, device=device) for s in ((4, 8), (16, 8), (16,)))
    a, m = fp8.quantize(x), fp8.quantize(w)
    for call in (lambda: fp8.quantize(x.int()), lambda: fp8.quantize(torch.zeros((), device=device)), lambda: fp8.quantize(x[:, :0]), lambda: fp8.quantize_columns(x[:0]),
                 lambda: fp8.quantize_both(x[:0]), lambda: fp8.dequantize(a, torch.int32), lambda: fp8.dequantize(a._replace(cols=200)), lambda: fp8.dequantize(a._replace(cols=0)),
                 lambda: fp8.dequantize(a._replace(scale=a.scale[:4])), lambda: fp8.dequantize(a._replace(q=a.q.view(torch.uint8))), lambda: fp8.scales(a._replace(cols=129)),
                 lambda: fp8.matmul(a, m._replace(cols=7)), lambda: fp8.matmul(a, m, b[:3]), lambda: fp8.matmul(a, m, b.to(BF), FP32), lambda: fp8.matmul(a, m, dtype=torch.int32),
                 lambda: fp8.linear(x[:, :5], w), lambda: fp8.linear(x, w[0]), lambda: fp8.linear(x, w, b[:5]), lambda: fp8.linear(x, w.to(BF)), lambda: fp8.linear(x, w, b.to(BF)),
                 lambda: fp8.linear(x.int(), w.int()), lambda: fp8.linear(x, w[:, :0]), lambda: fp8.linear(torch.zeros((), device=device), w),
                 lambda: fp8.linear(x[:, :5], m), lambda: fp8.linear(x, m, b[:5]), lambda: fp8.linear(x, m, b.to(BF)), lambda: fp8.linear(x.clone().requires_grad_(), m),
                 lambda: fp8.linear(x, m, b.clone().requires_grad_())):
        with pytest.raises(ValueError):
            call()
    with torch.no_grad():
        assert fp8.linear(x.clone().requires_grad_(), m).shape == (4, 16)


@pytest.mark.parametrize("device", DEVICES)
def test_second_derivatives_are_refused(device):
    x, w = torch.randn(4, 8, device=device).requires_grad_(), torch.randn(16, 8, device=device).requires_grad_()
    y = fp8.linear(x, w)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(y.sum(), (x, w), create_graph=True)


@pytest.mark.parametrize("device", DEVICES)
def test_forward_tangents_are_refused(device):
    """A result without a tangent would stand for a derivative of zero, and one through the rounding to 8 bits for a rounded derivative."""
    x, w, b = torch.randn(4, 200, device=device), torch.randn(16, 200, device=device), torch.randn(16, device=device)
    m = fp8.quantize(w)
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))      # noqa: E731
        for args in ((dual(x), w, b), (x, dual(w), b), (x, w, dual(b)), (dual(x), m, b), (x, m, dual(b))):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises((NotImplementedError, RuntimeError, ValueError)):
                    fp8.linear(*args)
        assert fwd.unpack_dual(fp8.dequantize(fp8.quantize(dual(x)))).tangent is None
        assert torch.equal(fp8.linear(x, m, b), fp8.linear(x, w, b))


def test_the_entry_points_refuse():
    """What no Python caller passes on: no launch comes of it."""
    assert lib.tmpi_fp8_quantize(16, 4, None, None, None, None, None, None, 4, 8, 7, None) != 0          # row pitch below the width, nothing to write
    assert lib.tmpi_fp8_quantize(16, 8, 16, 16, 16, None, None, None, 4, 8, 7, None) != 0                # a GELU along the rows alone
    assert lib.tmpi_fp8_quantize(16, 8, None, 8, 16, None, None, None, 4, 8, 7, None) != 0               # results at an odd address
    assert lib.tmpi_fp8_quantize(16, 8, None, 16, 16, None, None, None, 4, 8, 4, None) != 0              # integers
    assert lib.tmpi_fp8_few(16, 8, 16, 16, None, 16, 33, 4, 8, 0, 7, None) != 0
    assert lib.tmpi_fp8_product(16, 16, 16, 16, None, 16, None, 0, 4, 8, 0, 7, None, 0, None) != 0
    assert lib.tmpi_fp8_product(16, 16, 8, 16, None, 16, None, 4, 4, 8, 0, 7, None, 0, None) != 0
    assert lib.tmpi_fp8_product(16, 16, 16, 16, None, 16, 16, 4, 4, 8, 0, 7, None, 0, None) != 0         # a pre-activation without a GELU
    assert lib.tmpi_fp8_restore(8, 16, 16, 4, 8, 7, None) != 0 and lib.tmpi_fp8_restore(16, 16, 16, -1, 8, 7, None) != 0
    assert lib.tmpi_fp8_product_workspace_bytes(0, 4, 8) == 0
    assert lib.tmpi_fp8_product_sums(16, 16, 16, 16, 16, None, 1, 16, 4, 4, 8, 7, None, 0, None) != 0 and lib.tmpi_fp8_product_sums(16, 16, 16, 16, 16, 16, 0, 16, 4, 4, 8, 7, None, 0, None) != 0


@gpu
def test_refuses_tensors_of_two_devices_and_too_wide_ones():
    x, w, m = torch.zeros(4, 8), torch.zeros(16, 8), fp8.quantize(torch.zeros(16, 8))
    for call in (lambda: fp8.linear(x.cuda(), w), lambda: fp8.linear(x.cuda(), m), lambda: fp8.linear(x, fp8.quantize(w.cuda())), lambda: fp8.matmul(fp8.quantize(x.cuda()), m)):
        with pytest.raises(ValueError):
            call()
    ext, wide = _native.ext(), 2 ** 32 + 8
    new = lambda *s: torch.zeros(1, device="cuda").expand(s)      # noqa: E731
    assert ext.fp8_quantize(new(2, wide), True, False) is None and ext.fp8_linear(new(2, wide), new(3, wide), None, False) is None
    assert ext.fp8_linear(new(2, 8), new(wide, 8), None, False) is None


# ---------------------------------------------------------------- what a program meets
def _step(x, w, b, dy, gelu=True):
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    y = fp8.linear(*leaves, gelu=gelu)
    with torch.no_grad():
        few = fp8.linear(x[:5], fp8.quantize(w), b)
    return (y.detach(), few, *torch.autograd.grad(y, leaves, dy))


@gpu
def test_captured_step_with_other_inputs_and_another_stream():
    g = torch.Generator().manual_seed(10)
    new = lambda: [torch.randn(s, generator=g).to(BF).cuda() for s in ((260, 320), (136, 320), (136,), (260, 136))]      # noqa: E731
    sets = [new() for _ in range(3)]
    want = [_step(*s) for s in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s, v in zip(sets, want):
            assert all(torch.equal(a, b) for a, b in zip(_step(*s), v))
    torch.cuda.current_stream().wait_stream(side)
    held, graph = [t.clone() for t in sets[0]], torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(*held)
    for i in (0, 1, 2, 0):
        for h, t in zip(held, sets[i]):
            h.copy_(t)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, want[i])), i
    torch.cuda.synchronize()
    fp8.check_status()


@gpu
def test_two_streams_at_once():
    g = torch.Generator().manual_seed(11)
    s = [torch.randn(n, generator=g).to(BF).cuda() for n in ((1024, 1024), (1024, 1024), (1024,), (1024, 1024))]
    want = _step(*s)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for _ in range(4):
        for stream in streams:
            with torch.cuda.stream(stream):
                got.append(_step(*s))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for r in got for a, b in zip(r, want))


CAPTURE = '''
import sys, torch
from torchmpi_b200.ops import fp8
torch.manual_seed(0)
new = lambda *s: torch.randn(s, device="cuda").bfloat16().requires_grad_()
leaves, dy = [new(64, 128), new(256, 128), new(256)], torch.randn(64, 256, device="cuda").bfloat16()
forward = lambda: fp8.linear(*leaves, gelu=True)
def step():
    y = forward()
    if sys.argv[1] == "grad":
        return torch.autograd.grad(y, leaves, dy)
    y.backward(dy)
    return [t.grad for t in leaves]
side = torch.cuda.Stream()
side.wait_stream(torch.cuda.current_stream())
with torch.cuda.stream(side):
    step()
    alive = forward() if sys.argv[2] == "side" else None           # an eager graph of the same leaves
torch.cuda.current_stream().wait_stream(side)
alive = alive if alive is not None else forward()
for t in leaves:
    t.grad = None
with torch.cuda.stream(side):
    want = [g.clone() for g in torch.autograd.grad(forward(), leaves, dy)]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
try:
    with torch.cuda.graph(graph):
        got = step()
except RuntimeError:
    print("refused")
    sys.exit(0)
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, want))
print("as the eager step")
'''


@gpu
@pytest.mark.parametrize("where", ["side", "default"])
@pytest.mark.parametrize("how", ["grad", "backward"])
def test_captured_backward_while_an_eager_graph_lives(how, where):
    """In a process of its own, which has to survive.  Where the eager graph was made on the default stream, autograd refuses the capture with an exception for
    PyTorch's own operations as for these."""
    out = subprocess.run([sys.executable, "-c", CAPTURE, how, where], capture_output=True, text=True, timeout=300, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert out.returncode == 0 and ("as the eager step" in out.stdout or where == "default" and "refused" in out.stdout), out.stderr[-2000:]


@gpu
def test_more_elements_than_32_bits_count():
    """Matrices and results of more than 2^31 elements, at rows before and behind that border."""
    M, N, K = 70000, 32768, 128
    assert M * N > 2 ** 31
    g = torch.Generator(device="cuda").manual_seed(12)
    a, b = torch.randn(M, K, generator=g, device="cuda", dtype=BF), torch.randn(N, K, generator=g, device="cuda", dtype=BF)
    y = fp8.linear(a, fp8.quantize(b))
    rows = [0, 65534, 65535, 65536, 65537, M - 1]
    want, bound = ref.product(ref.kept(a[rows].cpu()), ref.kept(b.cpu()))
    ref.close(y[rows], want, bound + ref.half_step(want.abs() + bound, BF), "rows")
    m, t = fp8.quantize_both(y)                                              # [70000, 32768] and its transpose
    last = [0, 65536, M - 1]
    part = fp8.Block8(m.q[last].contiguous(), fp8._tiled(fp8.scales(m)[last]), N)
    assert torch.equal(fp8.dequantize(part, FP32).double().cpu(), ref.kept(y[last].cpu()))
    cols = [0, 30679, N - 1]
    part = fp8.Block8(t.q[cols].contiguous(), fp8._tiled(fp8.scales(t)[cols]), M)
    assert torch.equal(fp8.dequantize(part, FP32).double().cpu(), ref.kept(y[:, cols].t().cpu()))
    fp8.check_status()
