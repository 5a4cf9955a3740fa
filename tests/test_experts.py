"""Layers of experts: routing, rows to the experts and back, products grouped by expert, and the whole layer."""
import math
import os
import subprocess
import sys

import pytest
import torch

import expert_reference as ref
from torchmpi_b200 import _native
from torchmpi_b200.ops import act8, experts

gpu = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]
BF = torch.bfloat16


def _close32(got, want, terms=1):
    """fp32 results: a few roundings (2^-24 each) and a sum of `terms`; exp and the quotient are good to 2^-22."""
    off = (got.detach().double().cpu() - want).abs()
    ok = (off <= (8 + 2 * terms) * 2.0 ** -23 * (want.abs() + 1e-30) + 1e-12) | (torch.isnan(got.detach().cpu()) & torch.isnan(want))
    assert bool(ok.all()), float(off.nan_to_num(9e9).max())


# ---------------------------------------------------------------- routing
ROUTES = [(1, 1, 1), (1, 8, 2), (5, 3, 3), (16, 8, 2), (37, 64, 8), (200, 33, 4), (513, 5, 1), (257, 256, 32), (1000, 17, 6), (5000, 4, 2)]


def _logits(T, E, dtype, device, seed=0):
    """Coarse values (many ties), -0 beside 0, closed experts, tokens with no expert, with fewer than k, with NaN and infinity."""
    g = torch.Generator().manual_seed(seed)
    l = torch.randint(-6, 7, (T, E), generator=g).float() / 2
    l = torch.where(torch.rand(T, E, generator=g) < 0.1, torch.tensor(-0.0), l)
    l = torch.where(torch.rand(T, E, generator=g) < 0.15, -math.inf, l)
    if T > 4:
        l[1] = -math.inf
        l[2, 1:] = -math.inf
        l[3, 0] = math.nan
        l[4] = torch.finfo(dtype).min                      # a mask of the type's lowest value is an ordinary logit
    if T > 12:
        l[11] = math.nan
        l[12, E // 2] = math.inf
    return l.to(dtype).to(device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("T,E,k", ROUTES)
def test_route_is_the_definition(T, E, k, renormalize, device):
    for dtype in (torch.float32, BF, torch.float16):
        logits = _logits(T, E, dtype, device)
        r = experts.route(logits, k, renormalize)
        weights, chosen, order, place, offsets = ref.route(logits, k, renormalize)
        for got, want in ((r.chosen, chosen), (r.order, order), (r.place, place), (r.offsets, offsets)):
            assert got.dtype == torch.int32 and torch.equal(got.cpu().long(), want)
        _close32(r.weights, weights, E)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("T,E,k", ROUTES)
def test_route_gradient(T, E, k, renormalize, device):
    g = torch.Generator().manual_seed(2)
    logits = torch.randn(T, E, generator=g)
    logits = torch.where(torch.rand(T, E, generator=g) < 0.2, -math.inf, logits)
    logits[0, 0] = 0.5
    dw = torch.randn(T, k, generator=g)
    leaf = logits.to(device).requires_grad_(True)
    r = experts.route(leaf, k, renormalize)
    (got,) = torch.autograd.grad(r.weights, leaf, dw.to(device))
    weights, chosen, *_ = ref.route(logits, k, renormalize)
    wd = torch.where(chosen >= 0, weights * dw.double(), 0)
    mine = torch.zeros(T, E + 1, dtype=torch.float64).scatter_add_(1, torch.where(chosen >= 0, chosen, E), wd)[:, :E]
    p = torch.softmax(logits.double(), 1).nan_to_num(0)
    base = torch.zeros(T, E + 1, dtype=torch.float64).scatter_add_(1, torch.where(chosen >= 0, chosen, E), weights)[:, :E] if renormalize else p
    want = mine - base * wd.sum(1, keepdim=True)
    size = mine.abs() + base * wd.abs().sum(1, keepdim=True)
    assert bool(((got.cpu().double() - want).abs() <= (16 + 2 * E) * 2.0 ** -23 * size + 1e-12).all())


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("device", DEVICES)
def test_route_gradient_against_differences(device, renormalize):
    g = torch.Generator().manual_seed(4)
    T, E, k = 3, 6, 2
    logits, dw = torch.randn(T, E, generator=g), torch.randn(T, k, generator=g)
    leaf = logits.to(device).requires_grad_(True)
    (got,) = torch.autograd.grad(experts.route(leaf, k, renormalize).weights, leaf, dw.to(device))
    for t in range(T):
        for e in range(E):
            d = torch.zeros(T, E, dtype=torch.float64)
            d[t, e] = 1e-6
            up, down = (ref.route(logits.double() + s * d, k, renormalize)[0] for s in (1, -1))
            assert abs(float(((up - down) * dw.double()).sum() / 2e-6) - float(got[t, e])) < 1e-6


@gpu
def test_route_of_strided_logits():
    base = torch.randn(40, 64, device="cuda")
    for l in (base[:, :8], base[::2, 3:20], base.t(), base[:, ::2], base[:1, :8]):
        for a, b in zip(experts.route(l, 2), experts.route(l.contiguous(), 2)):
            assert torch.equal(a, b)
        leaf = l.detach().requires_grad_(True)
        dense = l.detach().contiguous().requires_grad_(True)
        dw = torch.randn(l.shape[0], 2, device="cuda")
        a, b = (torch.autograd.grad(experts.route(x, 2, False).weights, x, dw)[0] for x in (leaf, dense))
        assert torch.equal(a, b)


@gpu
def test_kernels_and_operations_agree_beyond_the_limits():
    for T, E, k in ((64, 300, 4), (40, 40, 33), (0, 8, 2)):
        logits = torch.randn(T, E, device="cuda")
        for a, b in zip(experts.route(logits, k)[1:], experts.route(logits.cpu(), k)[1:]):
            assert torch.equal(a.cpu(), b)


# ---------------------------------------------------------------- rows
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("T,E,k,C", [(1, 4, 1, 1), (6, 3, 2, 7), (50, 8, 2, 64), (33, 16, 5, 72), (300, 8, 8, 1000)])
def test_dispatch_and_combine(T, E, k, C, dtype, device):
    g = torch.Generator().manual_seed(6)
    half = torch.finfo(dtype).eps / 2
    x, dy = (torch.randn(T, C, generator=g).to(dtype).to(device) for _ in range(2))
    logits = torch.randn(T, E, generator=g)
    logits = torch.where(torch.rand(T, E, generator=g) < 0.3, -math.inf, logits)
    logits[0] = 0
    r = experts.route(logits.to(device), k)
    place, order, used = r.place.long(), r.order.long(), int(r.offsets[-1])
    x.requires_grad_(True)
    rows = experts.dispatch(x, r)
    want = torch.zeros(T * k, C, dtype=dtype, device=device)
    want[:used] = x.detach()[order[:used] // k]
    assert torch.equal(rows, want)
    drows = torch.randn(T * k, C, generator=g).to(dtype).to(device)
    (dx,) = torch.autograd.grad(rows, x, drows)
    picked = ref.V(torch.where((place >= 0).unsqueeze(2), drows.double()[place.clamp_min(0)], 0))
    ref.close(dx, ref.total(picked, 1).rounded(half), "dx")
    # and back
    rows = torch.randn(T * k, C, generator=g).to(dtype).to(device)
    rows[used:] = math.nan                                  # never read
    rows.requires_grad_(True)
    w = r.weights.detach().requires_grad_(True)
    y = experts.combine(rows, r._replace(weights=w))
    picked = torch.where((place >= 0).unsqueeze(2), rows.detach().double()[place.clamp_min(0)], 0)
    ref.close(y, ref.total(ref.mul(ref.V(w.detach().unsqueeze(2)), ref.V(picked)), 1).rounded(half), "y")
    dr, dw = torch.autograd.grad(y, (rows, w), dy)
    at = order[:used]
    ref.close(dr[:used], ref.mul(ref.V(w.detach().reshape(-1)[at].unsqueeze(1)), ref.V(dy[at // k])).rounded(half), "drows")
    assert not dr[used:].any()
    dots = ref.total(ref.mul(ref.V(dy.unsqueeze(1)), ref.V(picked)), 2)
    if device == "cpu":                                    # rows[used:] is NaN times zero there
        dots = ref.V(torch.where(place >= 0, dots.v, 0), dots.e)
    ref.close(dw, dots, "dweights")


# ---------------------------------------------------------------- products grouped by expert
def _offsets(sizes, device):
    return torch.tensor([0] + sizes).cumsum(0).int().to(device)


GROUPED = [
    # sizes of the groups, rows behind the last, K, N
    ([1], 0, 8, 8),
    ([3, 0, 1], 0, 64, 72),
    ([0, 0, 5, 0], 2, 40, 64),
    ([16] * 8, 0, 128, 256),
    ([33, 1, 31, 32, 64, 63, 65], 3, 72, 136),
    ([127, 128, 129, 0, 256, 255, 257], 0, 200, 320),
    ([300, 20], 130, 520, 1000),
    ([0, 700, 0, 0, 77], 1, 256, 512),
    ([5] * 40, 0, 64, 200),
    ([1] * 256, 7, 64, 64),
    ([0, 0], 9, 64, 64),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("gelu", [False, True])
@pytest.mark.parametrize("sizes,behind,K,N", GROUPED, ids=lambda v: str(v)[:24])
def test_grouped_linear(sizes, behind, K, N, gelu, device):
    g = torch.Generator().manual_seed(7)
    R, E = sum(sizes) + behind, len(sizes)
    dtype, half = (BF, ref.BF16) if device == "cuda" else (torch.float32, 2.0 ** -24)
    x, w, b = ref.grid(g, (R, K), 1 / 8, 2, device), ref.grid(g, (E, N, K), 1 / 64, 1 / 4, device), ref.grid(g, (E, N), 1 / 64, 1 / 2, device)
    dy = torch.randn(R, N, generator=g).to(device)
    if behind:
        x[R - behind:] = math.nan                          # rows of nobody: not read into any result
        dy[R - behind:] = math.inf
    x, w, b, dy = (t.to(dtype) for t in (x, w, b, dy))
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    launches = experts.launch_count
    y = experts.grouped_linear(*leaves, _offsets(sizes, device), gelu)
    got = (y, *torch.autograd.grad(y, leaves, dy))
    assert device == "cpu" or experts.launch_count >= launches + 3
    x, w, b = (t.detach() for t in leaves)
    zero = lambda *s: ref.V(torch.zeros(*s, dtype=torch.float64, device=device))
    want = (zero(R, N), zero(R, K), zero(E, N, K), zero(E, N))
    at = 0
    for e, n in enumerate(sizes):
        s = slice(at, at + n)
        at += n
        z = ref.V(x[s].double() @ w[e].double().t() + b[e].double())
        dz = ref.V(dy[s])
        out = z.rounded(half)
        if gelu:
            value = ref.gelu(z)[0]
            out, dz = value.rounded(half), ref.mul(dz, ref.gelu(z.rounded(half))[1]).rounded(half)
        for to, i, v in zip(want, (s, s, e, e), (out, ref.matmul(dz, ref.V(w[e])).rounded(half), ref.matmul(dz.t(), ref.V(x[s])).rounded(half),
                                                 ref.total(dz, 0).rounded(half))):
            to.v[i], to.e[i] = v.v, v.e
    for name, a, v in zip(("y", "dx", "dw", "db"), got, want):
        ref.close(a, v, name)
    with torch.no_grad():
        assert torch.equal(experts.grouped_linear(*leaves, _offsets(sizes, device), gelu), y)
    if device == "cuda":
        experts.check_status()


@gpu
def test_infinities_stay_with_their_expert():
    """An expert with infinite weights or rows leaves the results of the others as they are."""
    sizes, K, N = [70, 3, 90, 40], 72, 200
    x, w, dy = (torch.randn(s, device="cuda").to(BF) for s in ((203, K), (4, N, K), (203, N)))
    b = torch.randn(4, N, device="cuda").to(BF)
    off = _offsets(sizes, "cuda")

    def run(x, w, dy):
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
        y = experts.grouped_linear(*leaves, off)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))
    clean = run(x, w, dy)
    x2, w2, dy2 = x.clone(), w.clone(), dy.clone()
    x2[70:73], w2[1], dy2[70:73] = math.inf, math.nan, math.nan
    x2[163:], w2[3], dy2[163:] = math.nan, math.inf, -math.inf
    dirty = run(x2, w2, dy2)
    for rows in (slice(0, 70), slice(73, 163)):
        for i in (0, 1):
            assert torch.equal(clean[i][rows], dirty[i][rows])
    for e in (0, 2):
        for i in (2, 3):
            assert torch.equal(clean[i][e], dirty[i][e])


@gpu
def test_grouped_views_and_wanted_gradients():
    sizes, K, N = [40, 0, 33], 64, 72
    off = _offsets(sizes, "cuda")
    x, w, b, dy = (torch.randn(s, device="cuda").to(BF) for s in ((73, K), (3, N, K), (3, N), (73, N)))
    full = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = experts.grouped_linear(*full, off, True)
    want = torch.autograd.grad(y, full, dy)
    odd = lambda t: torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)       # an odd address
    views = [odd(x), w.transpose(1, 2).contiguous().transpose(1, 2), odd(b)]
    leaves = [t.requires_grad_(True) for t in views]
    y2 = experts.grouped_linear(*leaves, torch.stack([off, off], 1)[:, 0], True)
    assert torch.equal(y, y2)
    for a, c in zip(torch.autograd.grad(y2, leaves, dy.t().contiguous().t()), want):
        assert torch.equal(a, c)
    for wanted in ([0], [1], [2], [0, 2], [1, 2]):
        leaves = [t.clone().requires_grad_(i in wanted) for i, t in enumerate((x, w, b))]
        got = torch.autograd.grad(experts.grouped_linear(*leaves, off, True), [leaves[i] for i in wanted], dy)
        for i, a in zip(wanted, got):
            assert torch.equal(a, want[i])
    no_bias = experts.grouped_linear(x, w, None, off)
    assert torch.equal(no_bias, experts.grouped_linear(x, w, torch.zeros_like(b), off))


def test_grouped_gradient_against_differences():
    g = torch.Generator().manual_seed(8)
    sizes, K, N = [3, 0, 2], 5, 4
    leaves = [torch.randn(s, generator=g).requires_grad_(True) for s in ((6, K), (3, N, K), (3, N))]
    off, dy = _offsets(sizes, "cpu"), torch.randn(6, N, generator=g)
    y = experts.grouped_linear(*leaves, off, True)
    grads = torch.autograd.grad(y, leaves, dy)

    def f(x, w, b):
        s, at = 0.0, 0
        for e, n in enumerate(sizes):
            s = s + (torch.nn.functional.gelu(x[at:at + n] @ w[e].t() + b[e]) * dy[at:at + n].double()).sum()
            at += n
        return float(s)
    for i, grad in enumerate(grads):
        for at in range(0, grad.numel(), 2):
            p = [t.detach().double() for t in leaves]
            p[i].view(-1)[at] += 1e-5
            up = f(*p)
            p[i].view(-1)[at] -= 2e-5
            assert abs((up - f(*p)) / 2e-5 - float(grad.view(-1)[at])) < 2e-5


# ---------------------------------------------------------------- the layer
LAYERS = [(1, 4, 2, 8, 8), (4, 8, 2, 128, 256), (67, 5, 3, 72, 136), (300, 8, 2, 128, 512), (257, 16, 1, 264, 320), (33, 3, 3, 64, 96)]


def _layer_inputs(T, E, k, C, H, device, dtype=BF, seed=9):
    g = torch.Generator().manual_seed(seed)
    x, w1 = ref.grid(g, (T, C), 1 / 8, 2, device), ref.grid(g, (E, H, C), 1 / 64, 1 / 4, device)
    b1 = ref.grid(g, (E, H), 1 / 64, 1 / 2, device)
    w2, b2 = (torch.randn(E, C, H, generator=g) * H ** -0.5).to(device), (torch.randn(E, C, generator=g) * 0.1).to(device)
    dy, logits = torch.randn(T, C, generator=g).to(device), torch.randn(T, E, generator=g)
    logits = torch.where(torch.rand(T, E, generator=g) < 0.2, -math.inf, logits)
    logits[0] = 0.25
    return [t.to(dtype) for t in (x, w1, b1, w2, b2, dy)], logits.to(device)


NAMES = ("y", "dx", "dweights", "dw1", "db1", "dw2", "db2")


def _layer(inputs, logits, k, kept8):
    x, w1, b1, w2, b2, dy = inputs
    r = experts.route(logits, k)
    w = r.weights.detach().requires_grad_(True)
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, w1, b1, w2, b2)]
    y = experts.mlp(leaves[0], r._replace(weights=w), *leaves[1:], act8=kept8)
    dx, dw1, db1, dw2, db2, dwt = torch.autograd.grad(y, leaves + [w], dy)
    return r, (y.detach(), dx, dwt, dw1, db1, dw2, db2)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kept8", [False, True])
@pytest.mark.parametrize("T,E,k,C,H", LAYERS)
def test_layer(T, E, k, C, H, kept8, device):
    inputs, logits = _layer_inputs(T, E, k, C, H, device, BF if device == "cuda" else torch.float32)
    launches = experts.launch_count
    r, got = _layer(inputs, logits, k, kept8)
    assert device == "cpu" or experts.launch_count >= launches + 12
    x, w1, b1, w2, b2, dy = inputs
    for name, a, v in zip(NAMES, got, ref.experts(x, r.weights, r.chosen, w1, b1, w2, b2, dy, kept8)):
        ref.close(a, v, name)
    with torch.no_grad():
        assert torch.equal(experts.mlp(x, r, w1, b1, w2, b2, act8=kept8), got[0])
    assert all(torch.equal(a, b) for a, b in zip(_layer(inputs, logits, k, kept8)[1], got))
    if device == "cuda":
        experts.check_status()


@gpu
def test_layer_is_its_parts():
    """Route, dispatch, two grouped products and combine, one by one: the layer's formulas, with a rounding to bf16 between any two."""
    inputs, logits = _layer_inputs(190, 6, 2, 128, 256, "cuda")
    x, w1, b1, w2, b2, dy = inputs
    r = experts.route(logits, 2)
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, w1, b1, w2, b2)]
    w = r.weights.detach().requires_grad_(True)
    rw = r._replace(weights=w)
    h = experts.grouped_linear(experts.dispatch(leaves[0], r), leaves[1], leaves[2], r.offsets, gelu=True)
    y = experts.combine(experts.grouped_linear(h, leaves[3], leaves[4], r.offsets), rw)
    dx, dw1, db1, dw2, db2, dwt = torch.autograd.grad(y, leaves + [w], dy)
    for name, a, v in zip(NAMES, (y, dx, dwt, dw1, db1, dw2, db2), ref.experts(x, r.weights, r.chosen, w1, b1, w2, b2, dy, False, parts=True)):
        ref.close(a, v, name)


@gpu
def test_layer_without_biases_and_some_gradients():
    inputs, logits = _layer_inputs(61, 4, 2, 64, 128, "cuda")
    x, w1, b1, w2, b2, dy = inputs
    r = experts.route(logits, 2)
    zero = [torch.zeros_like(b1), torch.zeros_like(b2)]
    for kept8 in (False, True):
        assert torch.equal(experts.mlp(x, r, w1, None, w2, None, kept8), experts.mlp(x, r, w1, zero[0], w2, zero[1], kept8))
        _, want = _layer((x, w1, zero[0], w2, zero[1], dy), logits, 2, kept8)
        leaves = [t.clone().requires_grad_(True) for t in (x, w1, w2)]
        y = experts.mlp(leaves[0], r, leaves[1], None, leaves[2], None, kept8)
        for a, b in zip(torch.autograd.grad(y, leaves, dy), (want[1], want[3], want[5])):
            assert torch.equal(a, b)
        _, want = _layer(inputs, logits, 2, kept8)
        for i, at in enumerate((1, 3, 4, 5, 6)):
            leaves = [t.clone().requires_grad_(n == i) for n, t in enumerate((x, w1, b1, w2, b2))]
            y = experts.mlp(leaves[0], r, *leaves[1:], act8=kept8)
            assert torch.equal(torch.autograd.grad(y, leaves[i], dy)[0], want[at])


@gpu
def test_padding_tokens_are_left_alone():
    """Tokens without an expert give zeros, get no gradient, and change nothing for the others."""
    inputs, logits = _layer_inputs(90, 4, 2, 64, 128, "cuda")
    x, w1, b1, w2, b2, dy = inputs
    logits[60:] = -math.inf
    _, whole = _layer(inputs, logits, 2, True)
    x2, dy2 = x.clone(), dy.clone()
    x2[60:], dy2[60:] = math.nan, math.inf
    _, dirty = _layer((x2, w1, b1, w2, b2, dy2), logits, 2, True)
    r, alone = _layer((x[:60], w1, b1, w2, b2, dy[:60]), logits[:60], 2, True)
    want = ref.experts(x[:60], r.weights, r.chosen, w1, b1, w2, b2, dy[:60], True)
    assert not whole[0][60:].any() and not whole[1][60:].any() and not whole[2][60:].any()
    for name, a, b, c, v in zip(NAMES, whole, dirty, alone, want):
        n = 60 if a.shape[0] == 90 else a.shape[0]
        assert torch.equal(a[:n], b[:n]), name
        ref.close(a[:n], v, name)                          # a call of other sizes may add in another order
        ref.close(c, v, name)


@gpu
@pytest.mark.parametrize("kept8", [False, True])
def test_captured_step_with_other_logits(kept8):
    """One graph, replayed with tokens that go to other experts; and the same numbers on another stream."""
    (x, w1, b1, w2, b2, dy), logits = _layer_inputs(160, 6, 2, 64, 128, "cuda")
    sets = [(x, logits), (x.flip(0).contiguous(), logits.flip(1).contiguous()), (x, torch.where(torch.arange(6, device="cuda") == 3, logits.nan_to_num(0, 0, 0), -math.inf))]

    def step(x, l):
        leaves = [t.detach().requires_grad_(True) for t in (x, l, w1, b1, w2, b2)]
        r = experts.route(leaves[1], 2)
        y = experts.mlp(leaves[0], r, *leaves[2:], act8=kept8)
        return (y.detach(), r.offsets, *torch.autograd.grad(y, leaves, dy))
    want = [step(*s) for s in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s, w in zip(sets, want):
            assert all(torch.equal(a, b) for a, b in zip(step(*s), w))
    torch.cuda.current_stream().wait_stream(side)
    held, graph = [t.clone() for t in sets[0]], torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*held)
    for i in (0, 1, 2, 0):
        for h, t in zip(held, sets[i]):
            h.copy_(t)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, want[i])), i
    torch.cuda.synchronize()


@gpu
def test_two_streams_at_once():
    (x, w1, b1, w2, b2, dy), logits = _layer_inputs(300, 8, 2, 128, 256, "cuda")
    inputs = (x, w1, b1, w2, b2, dy)
    want = _layer(inputs, logits, 2, True)[1]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(4):
        for s, into in zip(streams, got):
            with torch.cuda.stream(s):
                into.append(_layer(inputs, logits, 2, True)[1])
    torch.cuda.synchronize()
    for results in got:
        for r in results:
            assert all(torch.equal(a, b) for a, b in zip(r, want))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kept8", [False, True])
def test_module(kept8, device):
    torch.manual_seed(0)
    m = experts.Experts(64, 128, 8, 2, act8=kept8).to(device).to(BF if device == "cuda" else torch.float32)
    x = torch.randn(2, 12, 64, device=device, dtype=m.w1.dtype, requires_grad=True)
    y = m(x)
    assert y.shape == x.shape and int(m.last_offsets[-1]) == 48
    y.float().square().sum().backward()
    assert all(p.grad is not None and p.grad.isfinite().all() and p.grad.any() for p in (*m.parameters(), x) if p is not m.b2 or True)


def test_refusals():
    x, w, b, off = torch.zeros(4, 8), torch.zeros(2, 16, 8), torch.zeros(2, 16), torch.tensor([0, 2, 4], dtype=torch.int32)
    r = experts.route(torch.randn(4, 2), 1)
    w2, b2 = torch.zeros(2, 8, 16), torch.zeros(2, 8)
    for call in (lambda: experts.route(torch.randn(4), 1), lambda: experts.route(torch.randn(4, 2), 3), lambda: experts.route(torch.randn(4, 2), 0),
                 lambda: experts.route(torch.ones(4, 2, dtype=torch.int32), 1),
                 lambda: experts.grouped_linear(x, w, b, off.long()), lambda: experts.grouped_linear(x, w, b, off[:2]),
                 lambda: experts.grouped_linear(x, w, b[:, :3], off), lambda: experts.grouped_linear(x[:, :4], w, b, off),
                 lambda: experts.grouped_linear(x, w.double(), None, off), lambda: experts.grouped_linear(x, w, b, torch.tensor([0, 3, 2], dtype=torch.int32)[[0, 1, 2]].flip(0)),
                 lambda: experts.dispatch(x[:3], r), lambda: experts.dispatch(x.int(), r), lambda: experts.combine(x[:3], r),
                 lambda: experts.dispatch(x, r._replace(order=r.order.long())), lambda: experts.combine(x, r._replace(weights=r.weights.double())),
                 lambda: experts.mlp(x, r, w, b, w2[:, :, :8], b2), lambda: experts.mlp(x[:3], r, w, b, w2, b2),
                 lambda: experts.mlp(x, r, w, b, w2.double(), b2), lambda: experts.mlp(x, r, torch.cat([w, w]), None, torch.cat([w2, w2]), None),
                 lambda: experts.Experts(8, 8, 2, 3)):
        with pytest.raises(ValueError):
            call()


@gpu
def test_refuses_tensors_of_two_devices():
    r = experts.route(torch.randn(4, 2, device="cuda"), 1)
    x, w, w2 = torch.zeros(4, 8), torch.zeros(2, 16, 8), torch.zeros(2, 8, 16)
    for call in (lambda: experts.dispatch(x, r), lambda: experts.combine(x, r), lambda: experts.mlp(x, r, w, None, w2, None),
                 lambda: experts.grouped_linear(x.cuda(), w, None, r.offsets), lambda: experts.grouped_linear(x, w, None, r.offsets)):
        with pytest.raises(ValueError):
            call()


@gpu
def test_wrong_offsets_stay_inside():
    """Offsets that descend, are negative or point behind the rows: the results mean nothing, and nothing outside is touched."""
    x, w, b = (torch.randn(s, device="cuda").to(BF) for s in ((50, 64), (3, 72, 64), (3, 72)))
    for bad in ([0, 40, 10, 50], [-5, 20, 30, 50], [0, 20, 90, 1 << 30], [7, 7, 7, 7], [50, 0, 50, 0]):
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
        y = experts.grouped_linear(*leaves, torch.tensor(bad, dtype=torch.int32, device="cuda"), True)
        torch.autograd.grad(y, leaves, torch.ones_like(y))
    torch.cuda.synchronize()
    experts.check_status()


# ---------------------------------------------------------------- what a training program meets
@gpu
@pytest.mark.parametrize("kept8", [False, True])
def test_no_tokens(kept8):
    x, w1, b1, w2, b2 = (t.requires_grad_() for t in (torch.empty(0, 8, device="cuda", dtype=BF), *(torch.randn(s, device="cuda").to(BF) for s in ((4, 16, 8), (4, 16), (4, 8, 16), (4, 8)))))
    y = experts.mlp(x, experts.route(torch.empty(0, 4, device="cuda"), 2), w1, b1, w2, b2, kept8)
    assert y.shape == (0, 8)
    for g, t in zip(torch.autograd.grad(y.sum(), (x, w1, b1, w2, b2)), (x, w1, b1, w2, b2)):
        assert g.shape == t.shape and bool((g == 0).all())


@gpu
@pytest.mark.parametrize("kept8", [False, True])
def test_saved_tensors_on_the_host_and_an_expanded_input(kept8):
    x, w1, b1, w2, b2 = leaves = [t.requires_grad_() for t in (torch.randn(1, 8, device="cuda").to(BF), *(torch.randn(s, device="cuda").to(BF) for s in ((4, 16, 8), (4, 16), (4, 8, 16), (4, 8))))]
    r = experts.route(torch.randn(6, 4, device="cuda"), 2)
    dy = torch.randn(6, 8, device="cuda").to(BF)
    grads = lambda y: torch.autograd.grad(y, leaves, dy)
    want = grads(experts.mlp(x.expand(6, 8).contiguous(), r, w1, b1, w2, b2, kept8))
    with torch.autograd.graph.save_on_cpu():
        y = experts.mlp(x.expand(6, 8), r, w1, b1, w2, b2, kept8)
    for a, b, c in zip(want, grads(y), grads(experts.mlp(x.expand(6, 8), r, w1, b1, w2, b2, kept8))):
        assert torch.equal(a, b) and torch.equal(a, c)


CAPTURE = '''
import sys, torch
from torchmpi_b200.ops import act8, experts
torch.manual_seed(0)
new = lambda *s: torch.randn(s, device="cuda").bfloat16().requires_grad_()
x, u1, u2, w1, w2 = new(64, 128), new(256, 128), new(128, 256), new(4, 256, 128), new(4, 128, 256)
logits, dy = torch.randn(64, 4, device="cuda", requires_grad=True), torch.randn(64, 128, device="cuda").bfloat16()
leaves = [x, u1, u2] if sys.argv[1] == "act8" else [x, logits, w1, w2]
forward = (lambda: act8.mlp(x, u1, None, u2, None)) if sys.argv[1] == "act8" else (lambda: experts.mlp(x, experts.route(logits, 2), w1, None, w2, None, act8=True))
def step():
    y = forward()
    if sys.argv[2] == "grad":
        return torch.autograd.grad(y, leaves, dy)
    y.backward(dy)
    return [t.grad for t in leaves]
side = torch.cuda.Stream()
side.wait_stream(torch.cuda.current_stream())
with torch.cuda.stream(side):
    step()
    alive = forward() if sys.argv[3] == "side" else None           # an eager graph of the same leaves
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
@pytest.mark.parametrize("what", ["act8", "experts"])
def test_captured_backward_while_an_eager_graph_lives(what, how, where):
    """In a process of its own, which has to survive.  Where the eager graph was made on the default stream, autograd refuses the capture with an
    exception for PyTorch's own operations as for these: a leaf's gradient belongs to the stream of the graph that met it first."""
    out = subprocess.run([sys.executable, "-c", CAPTURE, what, how, where], capture_output=True, text=True, timeout=300, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert out.returncode == 0 and ("as the eager step" in out.stdout or where == "default" and "refused" in out.stdout), out.stderr[-2000:]


@gpu
def test_more_elements_than_32_bits_count():
    """Both forms of the products, with results of more than 2^31 elements, against 64 bits at rows before and behind that border."""
    R, K, N = 600000, 64, 4096
    assert R * N > 2 ** 31
    x, w, off = torch.randn(R, K, device="cuda").to(BF), torch.randn(3, N, K, device="cuda").to(BF), torch.tensor([0, 10, R - 70, R - 5], dtype=torch.int32, device="cuda")
    groups = ((0, 3, 0), (10, 12, 1), (524286, 524290, 1), (R - 75, R - 70, 1), (R - 70, R - 5, 2))
    y = experts.grouped_linear(x, w, None, off)
    for a, b, e in groups:
        ref.close(y[a:b], ref.matmul(ref.V(x[a:b].cpu()), ref.V(w[e].cpu()).t()).rounded(), f"rows {a} to {b}")
    assert bool((y[R - 5:] == 0).all())
    dw, = torch.autograd.grad(experts.grouped_linear(x, w.requires_grad_(), None, off), w, y)
    ref.close(dw[2], ref.matmul(ref.V(y[R - 70:R - 5].cpu()).t(), ref.V(x[R - 70:R - 5].cpu())).rounded(), "dw of the last group")
    del x, y, dw
    R, N, E = 24000, 131072, 256
    assert R * N > 2 ** 31
    x, w, off = torch.randn(R, K, device="cuda").to(BF), torch.randn(E, N, K, device="cuda", dtype=BF), (torch.arange(E + 1, device="cuda") * R // E).int()
    y = experts.grouped_linear(x, w, None, off)
    for r in (0, 16383, 16384, R - 1):
        e = int((off <= r).sum()) - 1
        ref.close(y[r:r + 1], ref.matmul(ref.V(x[r:r + 1].cpu()), ref.V(w[e].cpu()).t()).rounded(), f"row {r}")
    experts.check_status()


@gpu
@pytest.mark.parametrize("kept8", [False, True])
@pytest.mark.parametrize("T,H", [(200, 40), (200, 72), (200, 128), (6, 40)])
def test_an_infinite_gradient_stays_infinite(T, H, kept8):
    """Positive weights, activations and a gradient with one infinity: the routing weight's gradient is infinite, not NaN, whatever lies behind the columns."""
    E, k, C = 2, 2, 16
    x, w1, w2 = (torch.rand(s, device="cuda").add(0.5).to(BF) for s in ((T, C), (E, H, C), (E, C, H)))
    r = experts.route(torch.zeros(T, E, device="cuda"), k)
    weights = r.weights.clone().requires_grad_()
    dy = torch.rand(T, C, device="cuda").add(0.5).to(BF)
    dy[T // 2, 3] = math.inf
    g, = torch.autograd.grad(experts.mlp(x, r._replace(weights=weights), w1, None, w2, None, kept8), weights, dy)
    inf = torch.zeros_like(g, dtype=torch.bool)
    inf[T // 2] = True
    assert torch.equal(torch.isinf(g) & (g > 0), inf) and not bool(torch.isnan(g).any())


@gpu
def test_widths_that_32_bits_do_not_count_are_left_to_pytorch():
    """A width of 2^32 + 8 is not one of 8: the kernels' entries take none of these (views of one element, nothing is allocated)."""
    ext, wide = _native.ext(), 2 ** 32 + 8
    new = lambda *s: torch.zeros(1, device="cuda", dtype=BF).expand(s)
    x, r = torch.zeros(4, 8, device="cuda", dtype=BF), experts.route(torch.zeros(4, 2, device="cuda"), 1)
    assert ext.grouped_linear(x, new(2, wide, 8), None, r.offsets, False) is None
    assert ext.grouped_linear(new(4, wide), new(2, 8, wide), None, r.offsets, False) is None
    assert ext.expert_mlp(x, *r, new(2, wide, 8), None, new(2, 8, wide), None, False) is None
    assert ext.act8_mlp(x, new(wide, 8), None, new(8, wide), None) is None
    assert ext.act8_mlp(x, new(8, 8), None, new(wide, 8), None) is None


@pytest.mark.parametrize("device", DEVICES)
def test_second_derivatives_are_refused(device):
    """A gradient asked for with a graph, which would be a constant in it, is refused."""
    new = lambda *s: torch.randn(s, device=device).to(BF).requires_grad_()
    x, w1, w2, u1, u2, logits = new(6, 16), new(4, 24, 16), new(4, 16, 24), new(24, 16), new(16, 24), torch.randn(6, 4, device=device, requires_grad=True)
    r = experts.route(logits.detach(), 2)
    calls = [(lambda: act8.mlp(x, u1, None, u2, None), (x, u1, u2)),
             (lambda: experts.mlp(x, experts.route(logits, 2), w1, None, w2, None, act8=True), (x, logits, w1, w2))]
    if device == "cuda":                      # elsewhere these are PyTorch's operations, which can be differentiated again
        calls += [(lambda: experts.mlp(x, r, w1, None, w2, None), (x, w1, w2)), (lambda: experts.route(logits, 2).weights, (logits,)),
                  (lambda: experts.dispatch(x, r), (x,)), (lambda: experts.combine(x.repeat(2, 1), r), (x,)),
                  (lambda: experts.grouped_linear(x, w1, None, torch.tensor([0, 2, 2, 5, 6], dtype=torch.int32, device=device)), (x, w1))]
    for call, leaves in calls:
        torch.autograd.grad(call().sum(), leaves)
        with pytest.raises(RuntimeError, match="once"):
            torch.autograd.grad(call().sum(), leaves, create_graph=True)
