"""8-bit activation checkpoints: the format, the GELU backward that reads one, and the MLP that keeps two."""
import math

import pytest
import torch

import expert_reference as ref
from torchmpi_b200.ops import act8, experts

gpu = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]
SHAPES = [(1, 1), (1, 8), (3, 31), (5, 32), (7, 33), (2, 40), (64, 96), (9, 1000), (130, 1024), (3, 5, 72)]
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _values(shape, dtype, device, seed=0):
    """Rows of very different sizes, ties of the rounding among them, zeros, subnormals, infinities and NaN."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp2(torch.randint(-12, 9, shape[:-1] + (1,), generator=g).float())
    ties = torch.randint(8, 16, shape, generator=g).float() * 2 + 1                 # half way between two e4m3 numbers
    x = torch.where(torch.rand(shape, generator=g) < 0.2, ties, x)
    x = torch.where(torch.rand(shape, generator=g) < 0.05, x * 2.0 ** -14, x)
    x = x.to(dtype)
    flat = x.view(-1)
    for i, v in enumerate((0.0, -0.0, math.inf, -math.inf, math.nan, torch.finfo(dtype).tiny / 4, 448.0, 449.0, -480.0, torch.finfo(dtype).max)):
        if flat.numel() > 40:
            flat[(i * 37) % flat.numel()] = v
    return x.to(device)


def _same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=1e30), torch.nan_to_num(b, nan=1e30))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_round_trip_is_the_definition(shape, dtype, device):
    x = _values(shape, dtype, device)
    a = act8.quantize(x)
    assert a.q.dtype == torch.float8_e4m3fn and a.q.shape == x.shape and a.scale.dtype == torch.uint8 and a.scale.shape == x.shape[:-1] + ((shape[-1] + 31) // 32,)
    for to in DTYPES:                    # exact but for what the type cannot hold: the largest fp32 numbers become 2^128, an infinity
        assert _same(act8.dequantize(a, to).cpu().float(), ref.kept(x.cpu()).to(to).float())


@pytest.mark.parametrize("device", DEVICES)
def test_error_is_half_a_step_of_e4m3(device):
    x = torch.randn(64, 256, device=device)
    off = (act8.dequantize(act8.quantize(x), torch.float32) - x).abs()
    top = x.view(64, 8, 32).abs().amax(2, keepdim=True).expand(64, 8, 32).reshape(64, 256)
    assert bool((off <= torch.maximum(x.abs() * 2.0 ** -4, top * 2.0 ** -10 / 224)).all())      # 224: the block's largest is at least that many units


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_views_and_odd_addresses(dtype):
    base = _values((66, 200), dtype, "cuda")
    for x in (base[:, 8:72], base[1:, 1:34], base.t(), base[:, ::2], base.view(-1)[3:3 + 64 * 96].view(64, 96)):
        a, b = act8.quantize(x), act8.quantize(x.contiguous().cpu())
        assert torch.equal(a.scale.cpu(), b.scale) and _same(a.q.cpu().float(), b.q.float())
        dy = torch.randn(x.shape, device="cuda").to(dtype)
        for got, want in zip(act8.gelu_gradient(dy, a), act8.gelu_gradient(dy.t().contiguous().t(), act8.Act8(a.q.clone(), a.scale.clone()))):
            assert _same(got.float(), want.float())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_gelu_gradient(shape, dtype, device):
    g = torch.Generator().manual_seed(3)
    x = (3 * torch.randn(shape, generator=g)).to(dtype)
    if x.numel() > 40:
        x.view(-1)[17] = math.nan
        x.view(-1)[23] = 400.0
        x.view(-1)[29] = -400.0
    dy = torch.randn(shape, generator=g).to(dtype).to(device)
    a = act8.quantize(x.to(device))
    h, slope = ref.gelu(ref.V(ref.kept(x).to(device)))
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * half                    # half a step of a subnormal result (fp16 has some here)
    dz, y = act8.gelu_gradient(dy, a)
    want = ref.mul(ref.V(dy), slope).rounded(half)
    ref.close(dz, ref.V(want.v, want.e + tiny), "dz")
    want = h.rounded(half)
    ref.close(y, ref.V(want.v, want.e + tiny), "h")


def test_gelu_gradient_against_differences():
    z = torch.arange(-40, 41).float().view(1, -1) / 8                   # multiples of 1/8 up to 5: each block's e4m3 numbers hold them to 2^-5 steps
    a = act8.quantize(z)
    z = act8.dequantize(a, torch.float64)
    f = lambda v: torch.nn.functional.gelu(v)
    slope = (f(z + 1e-5) - f(z - 1e-5)) / 2e-5
    dz, h = act8.gelu_gradient(torch.ones_like(z, dtype=torch.float32), a)
    assert (dz - slope).abs().max() < 1e-6 and (h - f(z)).abs().max() < 1e-6


MLPS = [(1, 8, 8, 8), (8, 128, 256, 128), (251, 64, 136, 72), (33, 520, 1000, 520), (300, 256, 512, 264), (1030, 128, 512, 128)]


def _mlp_inputs(T, C, H, D, device, dtype=torch.bfloat16, seed=5):
    g = torch.Generator().manual_seed(seed)
    x = ref.grid(g, (T, C), 1 / 8, 2, device)
    w1, b1 = ref.grid(g, (H, C), 1 / 64, 1 / 4, device), ref.grid(g, (H,), 1 / 64, 1 / 2, device)
    w2, b2 = (torch.randn(D, H, generator=g) * H ** -0.5).to(device), (torch.randn(D, generator=g) * 0.1).to(device)
    dy = torch.randn(T, D, generator=g).to(device)
    return [t.to(dtype) for t in (x, w1, b1, w2, b2, dy)]


@gpu
@pytest.mark.parametrize("T,C,H,D", MLPS)
def test_mlp_on_the_gpu(T, C, H, D):
    x, w1, b1, w2, b2, dy = _mlp_inputs(T, C, H, D, "cuda")
    leaves = [t.requires_grad_(True) for t in (x, w1, b1, w2, b2)]
    launches = act8.launch_count + experts.launch_count
    y = act8.mlp(*leaves)
    got = (y, *torch.autograd.grad(y, leaves, dy))
    assert act8.launch_count + experts.launch_count >= launches + 4      # both checkpoints' kernels and the grouped products'
    for name, a, b in zip(("y", "dx", "dw1", "db1", "dw2", "db2"), got, ref.mlp8(*[t.detach() for t in leaves], dy)):
        ref.close(a, b, name)
    with torch.no_grad():
        assert torch.equal(act8.mlp(*leaves), y)                        # without checkpoints the same numbers
    again = act8.mlp(*leaves)
    assert all(torch.equal(a, b) for a, b in zip((again, *torch.autograd.grad(again, leaves, dy)), got))


@gpu
def test_mlp_wanted_gradients_and_no_bias():
    x, w1, b1, w2, b2, dy = _mlp_inputs(40, 64, 128, 64, "cuda")
    full = [t.clone().requires_grad_(True) for t in (x, w1, b1, w2, b2)]
    want = dict(zip("xabcd", torch.autograd.grad(act8.mlp(*full), full, dy)))
    for wanted in ("x", "a", "b", "c", "d", "xc", "bd", "xb", "ab"):
        leaves = {n: t.clone().requires_grad_(n in wanted) for n, t in zip("xabcd", (x, w1, b1, w2, b2))}
        y = act8.mlp(*leaves.values())
        for n, got in zip(wanted, torch.autograd.grad(y, [leaves[n] for n in wanted], dy)):
            ref.close(got, ref.V(want[n], 2 * ref.BF16 * want[n].double().abs() + 1e-6 * dy.numel()), n)     # sums of another order
    zero = torch.zeros(64, device="cuda", dtype=torch.bfloat16)
    y0 = act8.mlp(x, w1, None, w2, None)
    assert torch.equal(y0, act8.mlp(x, w1, torch.zeros(128, device="cuda", dtype=torch.bfloat16), w2, zero))


@pytest.mark.parametrize("T,C,H,D", [(1, 8, 8, 8), (13, 5, 33, 7)])
def test_mlp_of_other_types(T, C, H, D):
    x, w1, b1, w2, b2, dy = _mlp_inputs(T, C, H, D, "cpu", torch.float32)
    leaves = [t.requires_grad_(True) for t in (x, w1, b1, w2, b2)]
    y = act8.mlp(*leaves)
    for name, a, b in zip(("y", "dx", "dw1", "db1", "dw2", "db2"), (y, *torch.autograd.grad(y, leaves, dy)), ref.mlp8(*[t.detach() for t in leaves], dy)):
        ref.close(a, b, name)


def test_mlp_against_differences():
    """Where the checkpoints are exact (small multiples), the gradient is that of the function itself."""
    g = torch.Generator().manual_seed(1)
    x, w1 = ref.grid(g, (6, 4), 1.0, 3, "cpu"), ref.grid(g, (9, 4), 1.0, 1, "cpu")          # |z| <= 12 in ones: four bits
    b1, w2, b2, dy = torch.zeros(9), torch.randn(3, 9, generator=g), torch.zeros(3), torch.randn(6, 3, generator=g)
    leaves = [t.float().requires_grad_(True) for t in (x, w1, b1, w2, b2)]
    grads = torch.autograd.grad(act8.mlp(*leaves), leaves, dy)
    f = lambda p: (torch.nn.functional.linear(torch.nn.functional.gelu(torch.nn.functional.linear(p[0], p[1], p[2])), p[3], p[4]) * dy.double()).sum()
    for i, grad in enumerate(grads):
        p = [t.detach().double() for t in leaves]
        for at in range(0, p[i].numel(), 3):
            d = torch.zeros_like(p[i]).view(-1)
            d[at] = 1e-5
            up, down = list(p), list(p)
            up[i], down[i] = p[i] + d.view_as(p[i]), p[i] - d.view_as(p[i])
            assert abs(float((f(up) - f(down)) / 2e-5) - float(grad.view(-1)[at])) < 1e-4


@gpu
def test_captured_step_and_another_stream():
    x, w1, b1, w2, b2, dy = _mlp_inputs(128, 64, 128, 64, "cuda")
    def step(x):
        leaves = [t.detach().requires_grad_(True) for t in (x, w1, b1, w2, b2)]
        y = act8.mlp(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))
    other = x.flip(0).contiguous()
    want = [step(x), step(other)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for a, b in zip(step(x), want[0]):
            assert torch.equal(a, b)
    torch.cuda.current_stream().wait_stream(side)
    held, graph = x.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(held)
    for given, expected in ((x, want[0]), (other, want[1]), (x, want[0])):
        held.copy_(given)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, expected))
    torch.cuda.synchronize()


@gpu
def test_keeps_less_memory():
    T, C, H = 2048, 256, 1024
    x, w1, b1, w2, b2, _ = _mlp_inputs(T, C, H, C, "cuda")
    leaves = [t.requires_grad_(True) for t in (x, w1, b1, w2, b2)]
    act8.mlp(*leaves)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = act8.mlp(*leaves)
    kept = torch.cuda.memory_allocated() - before - y.numel() * 2
    assert kept <= (T * (C + H)) * 33 // 32 + 8192


def test_empty_tensors():
    for shape in ((0, 32), (4, 0), (0,)):
        a = act8.quantize(torch.zeros(shape))
        assert act8.dequantize(a).shape == shape and a.scale.shape[-1] == (shape[-1] + 31) // 32
    w = torch.zeros(8, 8)
    assert act8.mlp(torch.zeros(0, 8), w, None, w, None).shape == (0, 8)


def test_refusals():
    x = torch.randn(4, 40)
    a = act8.quantize(x)
    for call in (lambda: act8.quantize(torch.zeros(4, 40, dtype=torch.int32)), lambda: act8.quantize(torch.tensor(1.0)),
                 lambda: act8.dequantize(act8.Act8(a.q, a.scale[:, :1])), lambda: act8.dequantize(act8.Act8(x, a.scale)),
                 lambda: act8.dequantize(act8.Act8(a.q, a.scale.float())), lambda: act8.dequantize(a, torch.int32),
                 lambda: act8.gelu_gradient(x[:, :39], a), lambda: act8.gelu_gradient(x.int(), a),
                 lambda: act8.mlp(x, torch.zeros(8, 32), None, torch.zeros(40, 8), None),
                 lambda: act8.mlp(x, torch.zeros(8, 40), torch.zeros(9), torch.zeros(40, 8), None),
                 lambda: act8.mlp(x, torch.zeros(8, 40).double(), None, torch.zeros(40, 8), None)):
        with pytest.raises(ValueError):
            call()


@gpu
def test_refuses_tensors_of_two_devices():
    x = torch.randn(4, 32)
    a = act8.quantize(x.cuda())
    for call in (lambda: act8.gelu_gradient(x, a), lambda: act8.dequantize(act8.Act8(a.q, a.scale.cpu())),
                 lambda: act8.mlp(x, torch.zeros(8, 32, device="cuda"), None, torch.zeros(8, 8), None)):
        with pytest.raises(ValueError):
            call()


# ---------------------------------------------------------------- what a training program meets
@gpu
def test_saved_tensors_on_the_host_and_an_expanded_input():
    x, w1, b1, w2, b2 = (t.requires_grad_() for t in _mlp_inputs(1, 40, 64, 24, "cuda")[:5])
    leaves = (x, w1, b1, w2, b2)
    dy = torch.randn(6, 24, device="cuda").bfloat16()
    grads = lambda y: torch.autograd.grad(y, leaves, dy)
    want = grads(act8.mlp(x.expand(6, 40).contiguous(), w1, b1, w2, b2))
    with torch.autograd.graph.save_on_cpu():
        y = act8.mlp(x.expand(6, 40), w1, b1, w2, b2)
    for a, b, c in zip(want, grads(y), grads(act8.mlp(x.expand(6, 40), w1, b1, w2, b2))):
        assert torch.equal(a, b) and torch.equal(a, c)


@gpu
def test_more_elements_than_32_bits_count():
    """The rows around and behind element 2^31 are those of small tensors (70000 x 32768, 4.6 GB)."""
    n, C = 70000, 32768
    x = torch.randn(n, C, device="cuda", dtype=torch.bfloat16)
    a = act8.quantize(x)
    y = act8.dequantize(a)
    rows = [0, 65535, 65536, n - 1]
    assert n * C > 2 ** 31
    for i in rows:
        assert _same(y[i].float().cpu(), ref.kept(x[i].cpu()).bfloat16().float())
    del y
    dz, h = act8.gelu_gradient(x, a)
    for i in rows:
        value, slope = ref.gelu(ref.V(ref.kept(x[i].cpu())))
        ref.close(h[i], value.rounded(), f"value of row {i}")
        ref.close(dz[i], ref.mul(ref.V(x[i].cpu()), slope).rounded(), f"gradient of row {i}")
