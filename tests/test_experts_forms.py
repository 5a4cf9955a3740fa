"""Every form of the products grouped by expert: which of them a call takes depends on its sizes, so the sizes here are chosen for the forms.

``few_mean`` rows to an expert (csrc/kernels/grouped.cu) are the border between the kernel with the weights as the rows of its MMAs and that on CTA pairs; with
more than 148 tiles, or 74 of a pair, a CTA has several one after the other.
"""
import math

import pytest
import torch

import expert_reference as ref
from torchmpi_b200._lib import lib
from torchmpi_b200.models import gpt2
from torchmpi_b200.ops import act8, experts, gemm

gpu = pytest.mark.gpu
BF = torch.bfloat16
NAMES = ("y", "dx", "dweights", "dw1", "db1", "dw2", "db2")


def _inputs(T, E, C, H, seed=9):
    """x w1^T + b1 is exact in fp32 (multiples of 1/512, below 2^15 of them)."""
    g = torch.Generator().manual_seed(seed)
    x, w1, b1 = ref.grid(g, (T, C), 1 / 8, 2, "cuda"), ref.grid(g, (E, H, C), 1 / 64, 1 / 4, "cuda"), ref.grid(g, (E, H), 1 / 64, 1 / 2, "cuda")
    w2, b2 = (torch.randn(E, C, H, generator=g) * H ** -0.5).cuda(), torch.randn(E, C, generator=g).cuda()
    dy, logits = torch.randn(T, C, generator=g).cuda(), torch.randn(T, E, generator=g)
    logits = torch.where(torch.rand(T, E, generator=g) < 0.2, -math.inf, logits)
    logits[0] = 0.25
    return [t.to(BF) for t in (x, w1, b1, w2, b2, dy)], logits.cuda()


def _layer(inputs, routing, kept8):
    x, w1, b1, w2, b2, dy = inputs
    w = routing.weights.detach().requires_grad_(True)
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, w1, b1, w2, b2)]
    y = experts.mlp(leaves[0], routing._replace(weights=w), *leaves[1:], act8=kept8)
    dx, dw1, db1, dw2, db2, dwt = torch.autograd.grad(y, leaves + [w], dy)
    return y.detach(), dx, dwt, dw1, db1, dw2, db2


def _check_layer(inputs, routing, kept8):
    x, w1, b1, w2, b2, dy = inputs
    got = _layer(inputs, routing, kept8)
    for name, a, v in zip(NAMES, got, ref.experts(x, routing.weights, routing.chosen, w1, b1, w2, b2, dy, kept8)):
        ref.close(a, v, name)
    with torch.no_grad():
        assert torch.equal(experts.mlp(x, routing, w1, b1, w2, b2, act8=kept8), got[0])
    assert all(torch.equal(a, b) for a, b in zip(_layer(inputs, routing, kept8), got))
    experts.check_status()


@gpu
@pytest.mark.parametrize("kept8", [False, True])
@pytest.mark.parametrize("T,E,k,C,H", [(512, 2, 2, 128, 256), (700, 4, 2, 136, 264), (331, 3, 1, 72, 200), (900, 5, 2, 200, 136), (257, 1, 1, 264, 64), (800, 6, 3, 8, 72)])
def test_fp32_results_of_the_kernel_on_pairs(T, E, k, C, H, kept8):
    """More than 96 rows to an expert: y and dx of a layer are fp32 results of the kernel on CTA pairs, added by combine.  Ragged groups, one of them empty, C no
    multiple of a tile's 64 columns among them."""
    inputs, logits = _inputs(T, E, C, H)
    if E > 2:
        logits[:, 1] = -math.inf
        logits[:, 2] -= 1.0
    r = experts.route(logits, k)
    assert T * k > 96 * E and lib.tmpi_grouped_slices(T * k, E, H, C) == 1
    _check_layer(inputs, r, kept8)


@gpu
@pytest.mark.parametrize("kept8", [False, True])
@pytest.mark.parametrize("T,H,parts", [(4, 1032, 2), (4, 1544, 3), (4, 2048, 4), (1, 4096, 4), (40, 4104, 4)])
def test_parts_of_k(T, H, parts, kept8):
    """Few rows and a long sum: an fp32 product is left in parts of K, the last one shorter, which combine adds; the bias is in the first alone."""
    E, k, C = 8, 2, 128
    inputs, logits = _inputs(T, E, C, H)
    r = experts.route(logits, k)
    assert lib.tmpi_grouped_slices(T * k, E, H, C) == parts
    _check_layer(inputs, r, kept8)


@gpu
@pytest.mark.parametrize("T,H", [(4100, 2056), (4100, 2048), (3001, 2600)])
def test_an_mlp_of_several_rounds(T, H):
    """More tiles than clusters, for the epilogues that keep the pre-activation in 8 bits and read it, with widths that are and are no multiple of 16 and 64."""
    C = D = 256
    assert -(-T // 256) * -(-H // 256) > 74
    (x, w1, b1, w2, b2, dy), _ = _inputs(T, 1, C, H)
    leaves = [t.requires_grad_(True) for t in (x, w1[0].contiguous(), b1[0].contiguous(), w2[0].contiguous(), b2[0].contiguous())]
    y = act8.mlp(*leaves)
    got = (y, *torch.autograd.grad(y, leaves, dy))
    for name, a, v in zip(("y", "dx", "dw1", "db1", "dw2", "db2"), got, ref.mlp8(*[t.detach() for t in leaves], dy)):
        ref.close(a, v, name)
    with torch.no_grad():
        assert torch.equal(act8.mlp(*leaves), y)
    experts.check_status()


@gpu
@pytest.mark.parametrize("kept8", [False, True])
@pytest.mark.parametrize("T,E,k,C,H", [(2000, 8, 2, 128, 1288), (2100, 7, 2, 64, 1536), (600, 128, 1, 64, 320), (450, 100, 2, 72, 392)])
def test_a_layer_of_several_rounds(T, E, k, C, H, kept8):
    """The same for a layer of experts: the kernel on pairs, and (128 and 100 experts) that for few rows.  Whole and partial tiles, and experts without rows."""
    inputs, logits = _inputs(T, E, C, H)
    logits[:, 3] = -math.inf
    logits[:, E - 1] += 1.5
    r = experts.route(logits, k)
    few = T * k <= 32 * E
    sizes = (r.offsets[1:] - r.offsets[:-1]).tolist()
    tile, columns, at_once = (128, 128, 148) if few else (256, 256, 74)
    assert sum(-(-n // tile) for n in sizes) * -(-H // columns) > at_once
    _check_layer(inputs, r, kept8)


@gpu
@pytest.mark.parametrize("sizes,behind,K,N", [([700, 0, 1300, 64, 1, 900, 31], 5, 72, 1288), ([333] * 12, 0, 64, 1024), ([9, 0, 40] * 40, 3, 72, 520)])
def test_a_gelu_of_several_rounds(sizes, behind, K, N):
    """grouped_linear with a GELU, with and without its pre-activation, and the backward pass."""
    g = torch.Generator().manual_seed(10)
    R, E = sum(sizes) + behind, len(sizes)
    x, w, b = ref.grid(g, (R, K), 1 / 8, 2, "cuda"), ref.grid(g, (E, N, K), 1 / 64, 1 / 4, "cuda"), ref.grid(g, (E, N), 1 / 64, 1 / 2, "cuda")
    dy = torch.randn(R, N, generator=g).cuda()
    x, w, b, dy = (t.to(BF) for t in (x, w, b, dy))
    off = torch.tensor([0] + sizes).cumsum(0).int().cuda()
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = experts.grouped_linear(*leaves, off, gelu=True)
    got = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        assert torch.equal(experts.grouped_linear(*leaves, off, gelu=True), y)
    x, w, b = (t.detach() for t in leaves)
    at = 0
    for e, n in enumerate(sizes):
        s = slice(at, at + n)
        at += n
        z = ref.V(x[s].double() @ w[e].double().t() + b[e].double())
        ref.close(y[s], ref.gelu(z)[0].rounded(), f"y of {e}")
        dz = ref.mul(ref.V(dy[s]), ref.gelu(z.rounded())[1]).rounded()
        for name, a, v in (("dx", got[0][s], ref.matmul(dz, ref.V(w[e]))), ("dw", got[1][e], ref.matmul(dz.t(), ref.V(x[s]))), ("db", got[2][e], ref.total(dz, 0))):
            ref.close(a, v.rounded(), f"{name} of {e}")
    assert not y[at:].any() and not got[0][at:].any()
    experts.check_status()


# ---------------------------------------------------------------- one rounding
def _exact_layer(T, H, seed=11):
    """Two experts, both of every token and with weights of one half, whose hidden values are whole numbers from 16 to 64 and equal, and whose second products nearly
    cancel.  A GELU is the identity there (1 - Phi(16) < 2^-150) and its slope 1, so every product and sum is one of a few bits and exact in fp32."""
    g = torch.Generator().manual_seed(seed)
    C = 24
    x = torch.randint(-1, 2, (T, C), generator=g).double()
    w1 = torch.randint(-1, 2, (1, H, C), generator=g).double().repeat(2, 1, 1)
    b1 = torch.full((2, H), 40.0, dtype=torch.float64)
    a = torch.randint(-127, 128, (C, H), generator=g).double() / 64
    w2 = torch.stack([a, torch.randint(-1, 2, (C, H), generator=g).double() / 64 - a])       # 8 bits each
    b2 = torch.randint(-64, 65, (2, C), generator=g).double() / 64
    return [t.cuda() for t in (x, w1, b1, w2, b2)]


@gpu
@pytest.mark.parametrize("kept8", [False, True])
@pytest.mark.parametrize("T,H", [(5, 64), (200, 64), (230, 72), (5, 1024), (30, 1032)])
def test_results_are_handed_over_in_fp32_and_rounded_once(T, H, kept8):
    """What experts return to a token, and the gradients that they return, are of many bits and nearly cancel: a rounding to bf16 before their sum would show."""
    x, w1, b1, w2, b2 = _exact_layer(T, H)
    dy = torch.zeros(T, x.shape[1], dtype=torch.float64)
    dy[torch.arange(T), torch.arange(T) * 7 % x.shape[1]] = 1.0                              # dy w2 is a row of w2: 8 bits
    dy = dy.cuda()
    r = experts.route(torch.zeros(T, 2, device="cuda"), 2)
    assert bool((r.weights == 0.5).all())
    z = x @ w1[0].t() + b1[0]
    h = z                                                                                    # forward: from the sums themselves
    y = 0.5 * (h @ w2[0].t() + b2[0]) + 0.5 * (h @ w2[1].t() + b2[1])
    zk = ref.kept(z) if kept8 else z                                                         # backward: from what is kept, whole numbers up to 64 again
    dh = torch.stack([dy @ w2[0], dy @ w2[1]])
    want = dict(y=y, dx=0.5 * (dh[0] + dh[1]) @ w1[0], dweights=torch.stack([(dh[e] * zk).sum(1) + dy @ b2[e] for e in range(2)], 1),
                dw1=torch.stack([0.5 * dh[e].t() @ x for e in range(2)]), db1=0.5 * dh.sum(1), dw2=(0.5 * dy.t() @ zk).expand(2, -1, -1), db2=(0.5 * dy.sum(0)).expand(2, -1))
    chosen = r.chosen.long()
    want["dweights"] = torch.gather(want["dweights"], 1, chosen)
    got = dict(zip(NAMES, _layer([t.to(BF) for t in (x, w1, b1, w2, b2, dy)], r, kept8)))
    for name in NAMES:
        if name == "dweights":                               # at most 60 additions one behind the other, and Phi good to 2^-22 of 1
            size = torch.gather(torch.stack([(dh[e] * zk).abs().sum(1) + dy.abs() @ b2[e].abs() for e in range(2)], 1), 1, chosen)
            assert bool(((got[name].double() - want[name]).abs() <= 64 * 2.0 ** -24 * size).all())
        else:
            assert torch.equal(got[name], want[name].to(torch.float32).to(BF)), name         # exact in fp32
    experts.check_status()


@gpu
@pytest.mark.parametrize("kept8", [False, True])
@pytest.mark.parametrize("T,H", [(5, 64), (200, 64), (230, 72)])
def test_a_routing_weights_gradient_is_added_from_fp32(T, H, kept8):
    """dweights = sum of (dy w2) h + dy . b2 with dy w2 of many bits: rounded to bf16 before the sum it would be off by 2^-13 of the sum of magnitudes and more."""
    x, w1, b1, w2, b2 = _exact_layer(T, H)
    g = torch.Generator().manual_seed(12)
    dy = torch.randint(-3, 4, x.shape, generator=g).double().cuda()
    r = experts.route(torch.zeros(T, 2, device="cuda"), 2)
    z = x @ w1[0].t() + b1[0]
    zk = ref.kept(z) if kept8 else z
    dh = torch.stack([dy @ w2[0], dy @ w2[1]])
    want = torch.gather(torch.stack([(dh[e] * zk).sum(1) + dy @ b2[e] for e in range(2)], 1), 1, r.chosen.long())
    size = torch.gather(torch.stack([(dh[e] * zk).abs().sum(1) + dy.abs() @ b2[e].abs() for e in range(2)], 1), 1, r.chosen.long())
    got = _layer([t.to(BF) for t in (x, w1, b1, w2, b2, dy)], r, kept8)[2].double()
    # in fp32, at most 60 additions one behind the other (16 and 2 in a slice of a row, a few for the slices, 13 for the bias), and Phi good to 2^-22 of 1
    assert bool(((got - want).abs() <= 64 * 2.0 ** -24 * size).all())
    rough = torch.gather(torch.stack([(dh[e].to(BF).double() * zk).sum(1) + dy @ b2[e] for e in range(2)], 1), 1, r.chosen.long())
    assert not bool(((rough - want).abs() <= 64 * 2.0 ** -24 * size).all())       # the bound tells the two apart


@gpu
@pytest.mark.parametrize("T", [5, 40, 300])
def test_a_hidden_gradient_is_rounded_once(T):
    """dz = (dy w2) gelu'(z~) in an MLP with 8-bit checkpoints: with one row of dy that is not zero the first bias's gradient is that row of dz, and it is within half a
    step of bf16 of the product of the fp32 sum and the slope; rounded twice, a part of them would not be."""
    C, H, D = 64, 512, 32
    g = torch.Generator().manual_seed(13)
    x, w1, b1 = ref.grid(g, (T, C), 1 / 8, 1, "cuda"), ref.grid(g, (H, C), 1 / 64, 1 / 8, "cuda"), ref.grid(g, (H,), 1 / 64, 1 / 2, "cuda")
    w2 = (torch.randint(-127, 128, (D, H), generator=g).double() / 64).cuda()
    dy = torch.zeros(T, D, dtype=torch.float64)
    dy[T // 2] = torch.randint(-3, 4, (D,), generator=g).double()
    dy = dy.cuda()
    leaves = [t.to(BF).requires_grad_(True) for t in (x, w1, b1, w2, torch.zeros(D, device="cuda"))]
    db1 = torch.autograd.grad(act8.mlp(*leaves), leaves[2], dy.to(BF))[0].double()
    z = ref.kept((x @ w1.t()).double() + b1.double())[T // 2]
    dh, slope = dy[T // 2] @ w2, torch.special.ndtr(z) + z * torch.exp(-z * z / 2) * 0.3989422804014327
    want, slack = dh * slope, dh.abs() * (1.6e-6 + 4e-7 * (1 + z.abs()))                      # of the slope: expert_reference.py
    half = torch.exp2(torch.floor(torch.log2((want.abs() + slack).clamp_min(1e-30))) - 8)     # half a step of eight bits
    assert bool(((db1 - want).abs() <= half + slack).all())
    twice = (dh.to(BF).double() * slope).to(BF).double()
    assert not bool(((twice - want).abs() <= half + slack).all())                             # the bound tells the two apart


# ---------------------------------------------------------------- the module with its gate, and what is left to PyTorch
@gpu
@pytest.mark.parametrize("kept8", [False, True])
@pytest.mark.parametrize("T", [24, 512])
def test_the_module_with_its_gate_against_64_bits(T, kept8):
    """The gradients through route, gate and experts together: the gate's weight, and the input, which has one from the experts and one through the gate."""
    E, k, C, H = 8, 2, 128, 256
    (x, w1, b1, w2, b2, dy), _ = _inputs(T, E, C, H)
    m = experts.Experts(C, H, E, k, act8=kept8).cuda().to(BF)
    g = torch.Generator().manual_seed(14)
    with torch.no_grad():
        for p, t in ((m.w1, w1), (m.b1, b1), (m.w2, w2), (m.b2, b2), (m.gate.weight, (torch.randn(E, C, generator=g) * C ** -0.5).to(BF))):
            p.copy_(t)
    x = x.requires_grad_(True)
    y = m(x)
    dx, dgate = torch.autograd.grad(y, (x, m.gate.weight), dy)
    x, gate = x.detach(), m.gate.weight.detach()
    logits = gemm.linear(x, gate).detach()
    r = experts.route(logits, k)
    want_y, dx_experts, dweights, *_ = ref.experts(x, r.weights, r.chosen, w1, b1, w2, b2, dy, kept8)
    ref.close(y, want_y, "y")
    chosen = r.chosen.long()
    p = torch.softmax(torch.gather(logits, 1, chosen).double(), 1)
    p = ref.V(p, 2.0 ** -21 * p)                              # an exponential, a sum and a quotient in fp32
    inner = ref.total(ref.mul(p, dweights), 1)
    parts = ref.mul(p, ref.add(dweights, ref.V(-inner.v.unsqueeze(1), inner.e.unsqueeze(1)))).rounded()
    dlogits = ref.V(torch.zeros(T, E, dtype=torch.float64, device="cuda").scatter_(1, chosen, parts.v), torch.zeros(T, E, dtype=torch.float64, device="cuda").scatter_(1, chosen, parts.e))
    ref.close(dgate, ref.matmul(dlogits.t(), ref.V(x)).rounded(), "dgate")
    ref.close(dx, ref.add(dx_experts, ref.matmul(dlogits, ref.V(gate)).rounded()).rounded(), "dx")
    assert dgate.any() and dlogits.v.abs().max() > 1e-2


@gpu
def test_a_blocks_input_gradient_with_the_gate():
    """The same inside a running model: what reaches the layer's input and its gate."""
    torch.manual_seed(4)
    net = gpt2.gpt2_tiny(n_layer=1, n_head=2, n_embd=128, block_size=128, vocab_size=512, tc_linear=True, n_expert=8).cuda().to(BF)
    m, held = net.blocks[0].experts, {}

    def look(module, args, out):
        held["x"] = args[0].detach()
        out.register_hook(lambda g: held.setdefault("dy", g.detach()))
        args[0].register_hook(lambda g: held.setdefault("dx", g.detach()))
    m.register_forward_hook(look)
    idx, target = torch.randint(0, 512, (2, 128), device="cuda"), torch.randint(0, 512, (2, 128), device="cuda")
    gpt2.LMLoss()(net(idx), target).backward()
    x = held["x"].clone().requires_grad_(True)
    dx, dgate = torch.autograd.grad(m(x), (x, m.gate.weight), held["dy"])
    assert torch.equal(dx, held["dx"]) and torch.equal(dgate, m.gate.weight.grad) and dgate.any()


@gpu
@pytest.mark.parametrize("kept8", [False, True])
@pytest.mark.parametrize("T,E,k,C,H", [(9, 3, 2, 12, 20), (130, 4, 1, 33, 65)])
def test_widths_that_the_kernels_do_not_take(T, E, k, C, H, kept8):
    """Widths that are no multiple of 8 run on PyTorch's operations: the same formulas, with the parts' roundings where nothing is kept in 8 bits."""
    inputs, logits = _inputs(T, E, C, H)
    r = experts.route(logits, k)
    x, w1, b1, w2, b2, dy = inputs
    for name, a, v in zip(NAMES, _layer(inputs, r, kept8), ref.experts(x, r.weights, r.chosen, w1, b1, w2, b2, dy, kept8, parts=not kept8)):
        ref.close(a, v, name)
