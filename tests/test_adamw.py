"""AdamW over many tensors, with states in 32 and 8 bits, and the norm of many gradients, against 64 bits."""
import math

import pytest
import torch

from torchmpi_b200._lib import lib
from torchmpi_b200.ops import adamw

gpu = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]
BF, HALF, FP32 = torch.bfloat16, torch.float16, torch.float32
SHAPES = [(7,), (128,), (130, 5), (1,), (300, 257), (0,), (2, 3, 1000), (4096,)]
LEAST = 2.0 ** -100


# ---------------------------------------------------------------- the definition in 64 bits
def _blocks(flat):
    return torch.nn.functional.pad(flat, (0, -flat.numel() % 128)).view(-1, 128)


def _codes(x, levels):
    """Codes in units (not rounded) of a block's elements, and the block's largest magnitude."""
    top = x.abs().amax(1, keepdim=True)
    return torch.sign(x) * levels * torch.sqrt(x.abs() / top.clamp_min(LEAST)), top


def _step(p, g, m, v, t, lr, betas, eps, decay, scale=1.0):
    b1, b2 = betas
    g = g * scale
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    p = p * (1 - lr * decay) - lr / (1 - b1 ** t) * m / (torch.sqrt(v / (1 - b2 ** t)) + eps)
    return p, m, v


def _make(shapes, dtype, device, seed=0, scale=0.05):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * scale).to(dtype).to(device).requires_grad_(True) for s in shapes]


def _grads(shapes, dtype, seed):
    g = torch.Generator().manual_seed(1000 + seed)
    return [(torch.randn(s, generator=g) * torch.exp(torch.randn(s, generator=g)) * 0.1).to(dtype) for s in shapes]


def _flat(opt, p, name):
    """A parameter's part of all moments or masters, as 64 bits in its shape."""
    return opt.state[p][name].double().cpu()


# ---------------------------------------------------------------- 32 bits
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype,master", [(FP32, True), (BF, True), (BF, False), (HALF, True), (HALF, False)])
@pytest.mark.parametrize("clip,scale", [(None, 1.0), (0.5, 1.0), (100.0, 0.25)])
def test_steps_of_32_bits(clip, scale, dtype, master, device):
    """Three steps, one of them without a gradient for a tensor.  Every number of a step is formed by a handful of fp32 operations: 2^-20 of the magnitudes that enter it."""
    ps = _make(SHAPES, dtype, device)
    groups = [{"params": ps[:3], "weight_decay": 0.1, "betas": (0.8, 0.95)}, {"params": ps[3:], "lr": 2e-2, "eps": 1e-6}]
    opt = adamw.AdamW(groups, lr=1e-2, master_weights=master, max_norm=clip, grad_scale=scale)
    w = [p.detach().double().cpu() for p in ps]
    m, v, t = [torch.zeros_like(x) for x in w], [torch.zeros_like(x) for x in w], [0] * len(w)
    launches = adamw.launch_count
    for i in range(3):
        grads = _grads(SHAPES, dtype, i)
        norm = 0.0
        for j, (p, g) in enumerate(zip(ps, grads)):
            p.grad = None if (i, j) == (1, 2) else g.to(device)
            norm += 0 if p.grad is None else float(g.double().square().sum())
        norm = abs(scale) * math.sqrt(norm)
        factor = scale * (min(1.0, clip / (norm + 1e-6)) if clip else 1.0)
        before = [p.detach().clone() for p in ps]
        opt.step()
        for j, p in enumerate(ps):
            if p.grad is None or not p.numel():
                assert torch.equal(p, before[j])
                continue
            t[j] += 1
            g = opt.param_groups[0 if j < 3 else 1]
            old = w[j]
            w[j], m[j], v[j] = _step(old, grads[j].double(), m[j], v[j], t[j], g["lr"], g["betas"], g["eps"], g["weight_decay"], factor)
            assert int(opt.state[p]["step"]) == t[j]
            off = 2.0 ** -20
            assert ((_flat(opt, p, "exp_avg") - m[j]).abs() <= off * (m[j].abs().amax() + 1e-30)).all()
            assert ((_flat(opt, p, "exp_avg_sq") - v[j]).abs() <= off * (v[j] + 1e-30)).all()
            step = off * (old.abs() + 20 * g["lr"])
            info = torch.finfo(dtype)
            if dtype != FP32 and master:
                assert ((_flat(opt, p, "master") - w[j]).abs() <= (i + 1) * step).all()
                assert torch.equal(p.detach(), opt.state[p]["master"].to(dtype))
            else:
                assert ((p.detach().double().cpu() - w[j]).abs() <= (i + 1) * step + w[j].abs() * info.eps / 2 + info.smallest_normal * info.eps).all()
                w[j] = p.detach().double().cpu()              # the next step goes by what was rounded
                if dtype != FP32:
                    assert "master" not in opt.state[p]
        if clip:
            assert float(opt.grad_norm) == pytest.approx(norm, rel=1e-6)
    assert device == "cpu" or adamw.launch_count - launches == (3 if clip is None else 6)


# ---------------------------------------------------------------- 8 bits
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype,master", [(FP32, True), (BF, True), (BF, False), (HALF, True)])
def test_steps_of_8_bits(dtype, master, device):
    """Each step from the states that the step before left: the averages are the nearest codes' (within a hundredth of a code of the border), the update is that of the averages before
    they were rounded."""
    ps = _make(SHAPES, dtype, device)
    opt = adamw.AdamW(ps, lr=1e-2, weight_decay=0.1, bits=8, master_weights=master, max_norm=3.0)
    for i in range(3):
        grads = _grads(SHAPES, dtype, i)
        norm = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
        state = [({k: x.clone().cpu() for k, x in opt.state[p].items()}, p.detach().double().cpu()) for p in ps]
        for p, g in zip(ps, grads):
            p.grad = g.to(device)
        opt.step()
        for p, g, (st, w) in zip(ps, grads, state):
            if not p.numel():
                continue
            n = p.numel()
            mc, vc = st["exp_avg"].double(), st["exp_avg_sq"].double()
            m0 = (torch.sign(mc) * (mc / 127) ** 2 * st["exp_avg_scale"].double().unsqueeze(1)).view(-1)[:n].view(p.shape)
            v0 = ((vc / 255) ** 4 * st["exp_avg_sq_scale"].double().unsqueeze(1) ** 2).view(-1)[:n].view(p.shape)
            if "master" in st:
                w = st["master"].double()
            want, m, v = _step(w, g.double(), m0, v0, i + 1, 1e-2, (0.9, 0.999), 1e-8, 0.1, min(1.0, 3.0 / (norm + 1e-6)))
            got = (opt.state[p]["master"] if "master" in st else p.detach()).double().cpu()
            info = torch.finfo(dtype if "master" not in st else FP32)
            assert ((got - want).abs() <= 2.0 ** -20 * (w.abs() + 0.2) + want.abs() * info.eps / 2 + info.smallest_normal * info.eps).all()
            for name, x, levels in (("exp_avg", m, 127), ("exp_avg_sq", v.sqrt(), 255)):
                code, top = _codes(_blocks(x.reshape(-1)), levels)
                if name == "exp_avg_sq":
                    code = torch.where(code > 0, code.clamp_min(1), 0)
                kept, scale = opt.state[p][name].double().cpu(), opt.state[p][name + "_scale"].double().cpu()
                assert ((kept - code).abs() <= 0.51).all(), name
                assert ((scale - top.view(-1)).abs() <= 2.0 ** -20 * top.view(-1)).all()
            mm, vv = opt.moments(p)
            unit = opt.state[p]["exp_avg_scale"].double().cpu().unsqueeze(1) / 127 ** 2
            c = opt.state[p]["exp_avg"].double().cpu()
            assert torch.allclose(_blocks(mm.double().cpu().reshape(-1)), c * c.abs() * unit, rtol=1e-6, atol=0)
            unit = opt.state[p]["exp_avg_sq_scale"].double().cpu().unsqueeze(1) / 255 ** 2
            c = opt.state[p]["exp_avg_sq"].double().cpu()
            assert torch.allclose(_blocks(vv.double().cpu().reshape(-1)), (c * c * unit) ** 2, rtol=1e-6, atol=0)
    whole = opt.moments()
    for i, p in enumerate(ps):
        for all_of, one in zip(whole, opt.moments(p)):
            assert all_of.dtype == BF and torch.equal(all_of[opt._places[i]: opt._places[i] + p.numel()], one.reshape(-1).to(BF))


@pytest.mark.parametrize("device", DEVICES)
def test_averages_without_gradients_shrink_alike(device):
    """The codes stay and the scales follow: nothing is lost in a thousand steps with gradients of zero."""
    p = torch.zeros(1000, device=device).requires_grad_(True)
    opt = adamw.AdamW([p], lr=0.0, bits=8, betas=(0.99, 0.999), weight_decay=0.0)
    p.grad = torch.randn(1000, generator=torch.Generator().manual_seed(3)).to(device)
    opt.step()
    first, code = [x.double().cpu() for x in opt.moments(p)], opt.state[p]["exp_avg"].clone()
    p.grad = torch.zeros_like(p)
    for _ in range(300):
        opt.step()
    assert torch.equal(opt.state[p]["exp_avg"], code) and not p.detach().any()
    for now, was, beta in zip(opt.moments(p), first, (0.99, 0.999)):
        assert torch.allclose(now.double().cpu(), was * beta ** 300, rtol=1e-4, atol=0)


@pytest.mark.parametrize("device", DEVICES)
def test_small_roots_do_not_become_zero(device):
    """One large gradient among tiny ones: the tiny ones' updates are smaller than with states of 32 bits, never larger."""
    g = torch.full((128,), 1e-7, device=device)
    g[5] = 10.0
    after = {}
    for bits in (8, 32):
        p = torch.zeros(128, device=device).requires_grad_(True)
        opt = adamw.AdamW([p], lr=1.0, bits=bits, weight_decay=0.0, eps=1e-12)
        for _ in range(3):
            p.grad = g.clone()
            opt.step()
        after[bits] = p.detach().abs()
        assert bits == 32 or (opt.state[p]["exp_avg_sq"] >= 1).all()
    assert (after[8] <= after[32] * 1.05).all() and after[8].isfinite().all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [8, 32])
def test_what_is_not_finite_shows(bits, device):
    """NaN and infinities reach the weight, in 8 bits those of their block of 128, and no other."""
    for bad in (math.nan, math.inf, -math.inf):
        p, q = (torch.ones(300, device=device).requires_grad_(True) for _ in range(2))
        opt = adamw.AdamW([p, q], bits=bits)
        for i in range(2):
            p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
            if i == 0:
                p.grad[130] = bad
            opt.step()
        lost = torch.zeros(300, dtype=torch.bool, device=device)
        lost[slice(128, 256) if bits == 8 else 130] = True
        assert torch.equal(torch.isnan(p.detach()), lost) and q.detach().isfinite().all()
        assert torch.isnan(opt.moments(p)[0]).sum() + torch.isinf(opt.moments(p)[0]).sum() == lost.sum()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [8, 32])
def test_no_gradient_no_eps(bits, device):
    """Elements that never had a gradient stay where they are, also with eps = 0, and the places behind a tensor's end stay zero."""
    p = torch.ones(200, device=device, dtype=BF).requires_grad_(True)
    opt = adamw.AdamW([p], eps=0.0, bits=bits, weight_decay=0.0, lr=0.5)
    p.grad = torch.zeros_like(p)
    p.grad[3] = 2.0
    opt.step()
    assert float(p.detach()[3]) == 0.5 and (p.detach()[4:] == 1).all() and (p.detach()[:3] == 1).all()
    assert not opt.moments()[0][200:].any() and not opt.moments()[1][200:].any() and not opt.masters()[200:].any()


# ---------------------------------------------------------------- layouts
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", [BF, FP32])
def test_strides_and_odd_addresses(bits, dtype, device):
    """Parameters and gradients at odd addresses, channels last, transposed, of other strides or types than their parameter: as if they lay as they should."""
    g = torch.Generator().manual_seed(4)
    values = [torch.randn(s, generator=g).to(dtype) for s in ((301,), (4, 8, 3, 3), (33, 20), (129,), (4, 8, 3, 3))]
    grads = [torch.randn(v.shape, generator=g).to(dtype) for v in values]

    def odd(t):
        room = torch.zeros(t.numel() + 3, dtype=dtype, device=device)
        room[3:] = t.reshape(-1).to(device)
        return room[3:].view(t.shape)
    last = torch.channels_last
    ps = [odd(values[0]), values[1].to(device).contiguous(memory_format=last), values[2].t().contiguous().t().to(device), values[3].to(device).clone(),
          values[4].to(device).contiguous(memory_format=last)]
    ps = [p.requires_grad_(True) for p in ps]
    plain = [v.to(device).clone().requires_grad_(True) for v in values]
    # in 8 bits the elements that share a scale follow each other in storage: the plain ones are laid out alike
    if bits == 8:
        plain[1], plain[2], plain[4] = (v.detach().contiguous(memory_format=last).requires_grad_(True) if v.dim() == 4 else v.detach().t().contiguous().t().requires_grad_(True)
                                        for v in (plain[1], plain[2], plain[4]))
    opts = [adamw.AdamW(x, lr=1e-2, bits=bits, max_norm=1.0) for x in (ps, plain)]
    for i in range(2):
        for a, b, v in zip(ps, plain, grads):
            b.grad = torch.empty_like(b).copy_(v.to(device) * (i + 1))
        ps[0].grad, ps[1].grad, ps[2].grad, ps[3].grad, ps[4].grad = (odd(grads[0] * (i + 1)), (grads[1] * (i + 1)).to(device), (grads[2] * (i + 1)).to(device),
                                                                     odd(grads[3] * (i + 1)), (grads[4] * (i + 1)).to(device).contiguous(memory_format=last))
        for o in opts:
            o.step()
    for a, b in zip(ps, plain):
        assert torch.equal(a, b)
        for x, y in zip(opts[0].moments(a), opts[1].moments(b)):
            assert x.shape == a.shape and torch.equal(x, y)


@gpu
@pytest.mark.parametrize("count", [99, 100, 101, 979, 981, 2100])
@pytest.mark.parametrize("bits", [8, 32])
def test_many_tensors(count, bits):
    """Tables of both sizes and several launches; the tensors of two types, every seventh without a gradient."""
    g = torch.Generator().manual_seed(count)
    sizes = torch.randint(1, 400, (count,), generator=g).tolist()
    make = lambda device: [torch.randn(n, generator=torch.Generator().manual_seed(i)).to(BF if i % 5 == 1 else FP32).to(device).requires_grad_(True) for i, n in enumerate(sizes)]      # noqa: E731
    a, b = make("cuda"), make("cpu")
    for ps in (a, b):
        for i, p in enumerate(ps):
            p.grad = None if i % 7 == 3 else torch.randn(p.shape, generator=torch.Generator().manual_seed(9 * i)).to(p.dtype).to(p.device)
    opts = [adamw.AdamW(ps, lr=1e-2, bits=bits, max_norm=2.0) for ps in (a, b)]
    for o in opts:
        o.step()
    assert float(opts[0].grad_norm) == pytest.approx(float(opts[1].grad_norm), rel=1e-6)
    assert torch.equal(opts[0]._steps.cpu(), opts[1]._steps)
    for x, y in zip(a, b):
        assert torch.allclose(x.detach().cpu().float(), y.detach().float(), rtol=1e-2 if x.dtype == BF else 1e-5, atol=1e-6)
    assert int(opts[0]._counter) == 0


@gpu
def test_a_tensor_of_more_than_32_bits_of_elements():
    """Its parts are further entries of one tensor: they take the same step count, and the states behind 2^31 are found."""
    n = 2 ** 31 + 2 ** 30 + 777
    p = torch.zeros(n, device="cuda", dtype=HALF).requires_grad_(True)
    p.grad = torch.zeros(n, device="cuda", dtype=HALF)
    places = [0, 2 ** 30 - 1, 2 ** 30, 2 ** 31 - 1, 2 ** 31, 2 ** 31 + 1, 2 ** 31 + 2 ** 30, n - 1]
    for i in places:
        p.grad[i] = 0.5
    opt = adamw.AdamW([p], lr=0.25, bits=8, master_weights=False, weight_decay=0.0, max_norm=1.0)
    for _ in range(2):
        opt.step()
    assert int(opt.state[p]["step"]) == 2 and float(opt.grad_norm) == pytest.approx(0.5 * len(places) ** 0.5, rel=1e-6)
    moved = torch.nonzero(p.detach()).view(-1).tolist()
    assert moved == places
    for i in places:
        assert float(p.detach()[i]) == pytest.approx(-0.5, rel=5e-3)


# ---------------------------------------------------------------- the norm
@pytest.mark.parametrize("device", DEVICES)
def test_norm(device):
    g = torch.Generator().manual_seed(5)
    for dtypes in ((FP32,), (BF,), (HALF, BF, FP32)):
        ts = [torch.randn(s, generator=g).to(dtypes[i % len(dtypes)]).to(device) for i, s in enumerate([(3,), (1000, 77), (0,), (5, 5), (2049,), (2048,), (1,)])]
        ts.append(ts[1][1:, 3:50])                                          # not dense
        ts.append(torch.randn(70001, generator=g).to(dtypes[0]).to(device)[1:])
        want = math.sqrt(sum(float(t.double().square().sum()) for t in ts))
        assert float(adamw.grad_norm(ts)) == pytest.approx(want, rel=1e-6)
        assert adamw.grad_norm(ts).shape == () and torch.equal(adamw.grad_norm(ts), adamw.grad_norm(ts))
    assert float(adamw.grad_norm([])) == 0 and float(adamw.grad_norm([torch.zeros(0, device=device)])) == 0
    assert math.isnan(float(adamw.grad_norm([torch.tensor([1.0, math.nan], device=device)]))) and math.isinf(float(adamw.grad_norm([torch.tensor([math.inf], device=device)])))
    assert float(adamw.grad_norm([torch.full((3,), 2.0, dtype=torch.float64, device=device)])) == pytest.approx(math.sqrt(12))


@pytest.mark.parametrize("device", DEVICES)
def test_a_norm_that_is_not_finite(device):
    """The coefficient is zero for an infinite norm and NaN for NaN, as the formula says: neither is hidden."""
    for bad in (math.inf, math.nan):
        p = torch.ones(10, device=device).requires_grad_(True)
        opt = adamw.AdamW([p], max_norm=1.0, weight_decay=0.0)
        p.grad = torch.ones_like(p)
        p.grad[2] = bad
        opt.step()
        assert torch.isnan(p.detach()[2]) and (math.isnan(float(opt.grad_norm)) or math.isinf(float(opt.grad_norm)))


# ---------------------------------------------------------------- a program
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [8, 32])
def test_state_dict(bits, device):
    def run(opt, ps, steps):
        for i in steps:
            for p, g in zip(ps, _grads(SHAPES, BF, i)):
                p.grad = g.to(device)
            opt.step()
    a = _make(SHAPES, BF, device)
    one = adamw.AdamW(a, lr=1e-2, bits=bits, max_norm=1.0)
    run(one, a, range(2))
    saved, weights = one.state_dict(), [p.detach().clone() for p in a]
    run(one, a, range(2, 4))
    b = [w.requires_grad_(True) for w in weights]
    two = adamw.AdamW(b, lr=5.0, bits=bits, max_norm=1.0)
    two.load_state_dict(saved)
    assert two.param_groups[0]["lr"] == 1e-2
    run(two, b, range(2, 4))
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and all(torch.equal(x, y) for x, y in zip(one.moments(), two.moments()))
    for broken in (dict(saved, bits=40 - bits), dict(saved, state=saved["state"][1:]), dict(saved, state=[dict(s, step=s["step"].long()) for s in saved["state"]]),
                   dict(saved, state=[{k: v for k, v in s.items() if k != "master"} for s in saved["state"]]), dict(saved, param_groups=saved["param_groups"] * 2)):
        with pytest.raises(ValueError):
            two.load_state_dict(broken)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [8, 32])
def test_checkpoint(bits, device, tmp_path):
    """A checkpoint file holds it beside the model; a resumed run takes the same steps."""
    from torchmpi_b200.utils import checkpoint

    def run(net, opt, steps):
        for i in steps:
            for p, g in zip(net.parameters(), _grads([q.shape for q in net.parameters()], BF, i)):
                p.grad = g.to(device)
            opt.step(1e-2)
    torch.manual_seed(0)
    a, b = (torch.nn.Linear(40, 30).to(BF).to(device) for _ in range(2))
    one, two = (adamw.AdamW(m.parameters(), bits=bits) for m in (a, b))
    run(a, one, range(2))
    checkpoint.save(str(tmp_path / "state.pt"), a, one)
    run(a, one, range(2, 4))
    checkpoint.load(str(tmp_path / "state.pt"), b, two)
    run(b, two, range(2, 4))
    assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters())) and torch.equal(one.masters(), two.masters())


@pytest.mark.parametrize("device", DEVICES)
def test_options_between_steps_and_refreshed_masters(device):
    p = torch.zeros(4, device=device, dtype=BF).requires_grad_(True)
    opt = adamw.AdamW([p], lr=1.0, weight_decay=0.0, eps=1e-6)
    p.grad = torch.ones_like(p)
    opt.step()
    assert torch.allclose(p.detach().float(), torch.full((4,), -1.0, device=device), rtol=1e-5)
    opt.step(lr=0.5)
    assert opt.param_groups[0]["lr"] == 0.5 and torch.allclose(p.detach().float(), torch.full((4,), -1.5, device=device), rtol=1e-5)
    opt.step(lr=torch.tensor(0.25, device=device))
    assert torch.allclose(p.detach().float(), torch.full((4,), -1.75, device=device), rtol=1e-5)
    with torch.no_grad():
        p.fill_(8)
    opt.refresh_master()
    opt.param_groups[0]["lr"] = 0.0
    version = p._version
    opt.step()
    assert (p == 8).all() and p._version > version
    opt.zero_grad(set_to_none=False)
    assert not p.grad.any()
    opt.zero_grad()
    assert p.grad is None
    opt.step()                                                               # nothing to do


@gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_captured_step(bits):
    """A replayed step counts on, with the rate that lies on the device and the gradients of the replay; the eager steps of another optimizer go on meanwhile."""
    shapes = SHAPES + [(50,)] * 120
    a, b = _make(shapes, BF, "cuda"), _make(shapes, BF, "cuda")
    rate = torch.tensor(1e-2, device="cuda")
    one, two = adamw.AdamW(a, lr=rate, bits=bits, max_norm=1.0), adamw.AdamW(b, lr=1e-2, bits=bits, max_norm=1.0)
    for p in a:
        p.grad = torch.zeros_like(p)
    graph = torch.cuda.CUDAGraph()
    before = [p.detach().clone() for p in a]
    with torch.cuda.graph(graph):
        one.step()
    assert all(torch.equal(x, y) for x, y in zip(a, before))
    for i in range(3):
        rate.fill_(1e-2 / (i + 1))
        for p, q, g in zip(a, b, _grads(shapes, BF, i)):
            p.grad.copy_(g)
            q.grad = g.cuda()
        graph.replay()
        two.step(lr=float(rate))
        assert torch.equal(one._steps, two._steps)
        for p, q in zip(a, b):
            assert torch.equal(p, q)
    torch.cuda.synchronize()


@gpu
def test_another_stream_and_two_optimizers_at_once():
    want = None
    for streams in (None, [torch.cuda.Stream(), torch.cuda.Stream()]):
        sets = [_make([(500, 300), (77,)], BF, "cuda", seed=s) for s in range(2)]
        opts = [adamw.AdamW(ps, lr=1e-2, bits=8, max_norm=1.0) for ps in sets]
        for ps in sets:
            for p in ps:
                p.grad = torch.ones_like(p)
        torch.cuda.synchronize()
        for _ in range(20):
            for i, o in enumerate(opts):
                with torch.cuda.stream(streams[i] if streams else torch.cuda.current_stream()):
                    o.step()
        torch.cuda.synchronize()
        got = [p.detach() for ps in sets for p in ps]
        want = want or got
        assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    p = torch.zeros(4, 6, device=device)
    new = lambda *s, **k: torch.zeros(*s, device=device, **k).requires_grad_(True)      # noqa: E731
    for call in (lambda: adamw.AdamW([]), lambda: adamw.AdamW([p], bits=16), lambda: adamw.AdamW([p], max_norm=0.0), lambda: adamw.AdamW([p], betas=(0.9, 1.0)),
                 lambda: adamw.AdamW([p], betas=(-0.1, 0.9)), lambda: adamw.AdamW([p], lr=-1.0), lambda: adamw.AdamW([p], eps=-1.0), lambda: adamw.AdamW([p], weight_decay=-1.0),
                 lambda: adamw.AdamW([p, p]), lambda: adamw.AdamW([{"params": [p], "momentum": 0.9}]), lambda: adamw.AdamW([p.double()]), lambda: adamw.AdamW([p.int()]),
                 lambda: adamw.AdamW([p[:, :3]]), lambda: adamw.AdamW([torch.zeros(1, device=device).expand(5)]), lambda: adamw.AdamW([new(3) * 2]),
                 lambda: adamw.AdamW([{"params": [torch.zeros(1, device=device)]} for _ in range(9)]), lambda: adamw.grad_norm([p.int()])):
        with pytest.raises(ValueError):
            call()
    q = new(4, 6)
    opt = adamw.AdamW([q])
    opt.param_groups[0]["betas"] = (0.9, 2.0)
    q.grad = torch.zeros_like(q)
    with pytest.raises(ValueError):
        opt.step()
    assert int(opt.state[q]["step"]) == 0


@gpu
def test_refuses_what_has_moved():
    q = torch.zeros(4, 6, device="cuda").requires_grad_(True)
    opt = adamw.AdamW([q])
    q.grad = torch.zeros_like(q)
    for data in (torch.zeros(4, 7, device="cuda"), torch.zeros(4, 12, device="cuda")[:, ::2], torch.zeros(4, 6)):
        q.grad = None
        q.data = data
        q.grad = torch.zeros_like(q)
        with pytest.raises(ValueError):
            opt.step()
    with pytest.raises(ValueError):
        adamw.AdamW([torch.zeros(3, device="cuda"), torch.zeros(3)])
    q = torch.zeros(4, 6, device="cuda").requires_grad_(True)
    opt = adamw.AdamW([q])
    q.grad = torch.zeros_like(q)
    with pytest.raises(ValueError):
        opt.step(lr=torch.tensor(0.1))
    assert int(opt.state[q]["step"]) == 0


@pytest.mark.parametrize("device", DEVICES)
def test_a_loaded_learning_rate_lies_where_it_lay(device):
    """On the parameters' device, and in the tensor that a captured step reads, wherever the saved one lies."""
    made = lambda lr: adamw.AdamW([torch.zeros(5, device=device).requires_grad_(True)], lr=lr)      # noqa: E731
    saved = made(torch.tensor(0.25, device=device)).state_dict()
    saved["param_groups"][0]["lr"] = saved["param_groups"][0]["lr"].cpu()
    rate = torch.tensor(0.5, device=device)
    for opt in (made(rate), made(0.5)):
        opt.load_state_dict(saved)
        lr = opt.param_groups[0]["lr"]
        assert lr.device == rate.device and float(lr) == 0.25 and lr is not saved["param_groups"][0]["lr"]
        p = next(iter(opt.state))
        p.grad = torch.ones_like(p)
        opt.step()
        assert torch.allclose(p.detach(), torch.full_like(p, -0.25), rtol=1e-6)          # the first step has the rate's length
    assert float(rate) == 0.25


@pytest.mark.parametrize("device", DEVICES)
def test_refuses_another_order_or_type_of_a_parameter(device):
    """The states lie in the order that the parameter had: in another they would be those of other elements."""
    for change in (lambda q: q.data.t().contiguous().t(), lambda q: q.data.bfloat16(), lambda q: q.data.reshape(6, 4)):
        q = torch.randn(4, 6, device=device).requires_grad_(True)
        before = torch.randn(3, device=device).requires_grad_(True)
        opt = adamw.AdamW([q, before])
        q.data = change(q)
        q.grad = torch.zeros_like(q)
        with pytest.raises(ValueError):
            opt.step()
        assert int(opt.state[q]["step"]) == 0
    q = torch.randn(1, 6, device=device).requires_grad_(True)          # a dimension of one element has no order
    opt = adamw.AdamW([q])
    q.data = torch.randn(6, 1, device=device).t()
    q.grad = torch.ones_like(q)
    opt.step()
    assert int(opt.state[q]["step"]) == 1


def test_the_entry_points_refuse():
    """What no Python caller passes on: no launch comes of it."""
    assert lib.tmpi_adamw_max_groups() == 8
    assert lib.tmpi_adamw_values(8, 16, 16, 16, 16, 16, 1, 7, None) != 0 and lib.tmpi_adamw_values(16, 16, 16, 16, 16, 16, -1, 7, None) != 0
    assert lib.tmpi_norm_squares(None, -1, 7, None, (__import__("ctypes").c_int * 1)(), None, None) != 0


@gpu
def test_64_bits_of_norms_and_mixed_devices():
    a = torch.ones(5, device="cuda")
    with pytest.raises(ValueError):
        adamw.grad_norm([a, torch.ones(5)])
    assert adamw.grad_norm([a.double()]).dtype == torch.float64


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [8, 32])
def test_a_refused_step_changes_nothing(bits, device):
    """The last of the parameters is refused, and the first ones, the counts, the averages and the norm are as they were."""
    p = [torch.ones(300, device=device), torch.ones(5, 7, device=device)]
    o = adamw.AdamW(p, bits=bits, max_norm=1.0)
    for t in p:
        t.grad = torch.full_like(t, 0.5)
    o.step()
    p[1].grad = None
    p[1].data = p[1].data.t()
    p[1].grad = torch.full_like(p[1], 2.0)
    before = [t.clone() for t in (p[0], o.state[p[0]]["step"], *o.moments(), o.grad_norm)]
    with pytest.raises(ValueError, match="changed"):
        o.step()
    assert all(torch.equal(a, b) for a, b in zip(before, (p[0], o.state[p[0]]["step"], *o.moments(), o.grad_norm)))
