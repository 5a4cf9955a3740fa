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


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype,grad_dtype,master", [(BF, FP32, True), (BF, FP32, False), (HALF, FP32, True), (HALF, FP32, False), (HALF, BF, True), (BF, HALF, False), (FP32, BF, True)])
def test_gradients_of_another_type(dtype, grad_dtype, master, bits, device):
    """A gradient counts as it is, not rounded to its parameter's type: 1 + 2^-12 is not 1, and what fp16 does not hold is not infinite.  Beside parameters with gradients of their own
    type, transposed ones among them."""
    gen = torch.Generator().manual_seed(6)
    shapes = [(33, 20), (300,), (129,)]
    ps = [torch.randn(s, generator=gen).to(dtype).to(device) for s in shapes]
    ps[0] = ps[0].t().contiguous().t()
    ps = [p.requires_grad_(True) for p in ps]
    opt = adamw.AdamW(ps, lr=1e-2, weight_decay=0.1, eps=1e-6, bits=bits, master_weights=master, max_norm=1e9)
    grads = [torch.randn(s, generator=gen) for s in shapes]
    grads[1][:4] = torch.tensor([1 + 2.0 ** -12, 1e5 if dtype == HALF else 1.0, -(1 + 2.0 ** -9), 2.0 ** -10])
    grads[1] = grads[1].to(grad_dtype)
    grads[0], grads[2] = grads[0].to(grad_dtype), grads[2].to(dtype)
    old = [p.detach().double().cpu() for p in ps]
    for p, g in zip(ps, grads):
        p.grad_dtype = None
        p.grad = g.to(device)
    version = ps[1]._version
    opt.step()
    assert ps[1]._version > version
    want_norm = sum(float(g.double().square().sum()) for g in grads) ** 0.5
    assert float(opt.grad_norm) == pytest.approx(want_norm, rel=1e-6)
    for p, g, w in zip(ps, grads, old):
        g = g.double()
        m, v = 0.1 * g, 0.001 * g * g
        want = w * (1 - 1e-3) - 1e-2 * g / (g.abs() + 1e-6)
        info = torch.finfo(dtype)
        assert int(opt.state[p]["step"]) == 1
        if "master" in opt.state[p]:
            assert ((opt.state[p]["master"].double().cpu() - want).abs() <= 2.0 ** -20 * (w.abs() + 0.2)).all()
            assert torch.equal(p.detach(), opt.state[p]["master"].to(dtype))
        assert ((p.detach().double().cpu() - want).abs() <= 2.0 ** -20 * (w.abs() + 0.2) + want.abs() * info.eps / 2 + info.smallest_normal * info.eps).all()
        if bits == 32:
            for got, x in zip(opt.moments(p), (m, v)):
                assert ((got.double().cpu() - x).abs() <= 2.0 ** -20 * x.abs() + 1e-30).all()
        else:
            top = opt.state[p]["exp_avg_scale"].double().cpu()
            flat = torch.empty_strided(p.shape, p.stride(), dtype=torch.float64).copy_(m).as_strided((p.numel(),), (1,))
            pieces = torch.nn.functional.pad(flat, (0, -p.numel() % 128)).view(-1, 128).abs().amax(1)
            assert ((top - pieces).abs() <= 2.0 ** -20 * pieces).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("master", [True, False])
def test_states_of_another_order(master, bits, device):
    """Codes of 8 bits lie in the order of the parameter's storage: in another order, or of another shape, they are refused and nothing changes.  States of 32 bits are those of the elements."""
    last = torch.channels_last

    def made(memory_format, shape=(8, 16, 3, 3)):
        p = torch.randn(shape, generator=torch.Generator().manual_seed(1)).to(BF).to(device).contiguous(memory_format=memory_format).requires_grad_(True)
        return p, adamw.AdamW([p], lr=1e-2, bits=bits, master_weights=master)
    p, one = made(last)
    p.grad = torch.randn(p.shape, generator=torch.Generator().manual_seed(2)).to(BF).to(device)
    one.step()
    saved = one.state_dict()
    q, same = made(last)
    same.load_state_dict(saved)
    assert all(torch.equal(a, b) for a, b in zip(one.moments(p), same.moments(q)))
    others = [made(torch.contiguous_format)]
    if not (bits == 32 or master):                       # by their codes alone they could be another shape's
        others.append(made(last, (16, 8, 3, 3)))
    for q, other in others:
        if bits == 8:
            before = [t.clone() for t in (*other.moments(), other.state[q]["step"])]
            with pytest.raises(ValueError, match="order"):
                other.load_state_dict(saved)
            assert all(torch.equal(a, b) for a, b in zip(before, (*other.moments(), other.state[q]["step"])))
        else:
            other.load_state_dict(saved)
            assert all(torch.equal(a, b) for a, b in zip(one.moments(p), other.moments(q)))
    saved.pop("layout", None)                            # a state without it is taken for one of the same order
    q, same = made(last)
    same.load_state_dict(saved)
    assert all(torch.equal(a, b) for a, b in zip(one.moments(p), same.moments(q)))
    one_row, saved = torch.zeros(6, 1, device=device).t().requires_grad_(True), None          # a dimension of one element has no order
    a, b = adamw.AdamW([one_row], bits=bits), adamw.AdamW([torch.zeros(1, 6, device=device).requires_grad_(True)], bits=bits)
    b.load_state_dict(a.state_dict())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("options", [dict(lr=-1.0), dict(betas=(0.9, 2.0)), dict(eps=-1.0), dict(weight_decay=-1.0), dict(eps=torch.tensor(0.1)), dict(lr=torch.tensor([0.1, 0.2])),
                                     dict(betas=0.9)], ids=str)
def test_options_that_are_none_are_not_loaded(options, device):
    """Refused before anything has changed, the options of the groups before and the averages among it."""
    ps = [torch.ones(5, device=device).requires_grad_(True) for _ in range(2)]
    rate = torch.tensor(0.5, device=device)
    opt = adamw.AdamW([{"params": ps[:1], "lr": 0.25}, {"params": ps[1:], "lr": rate}])
    for p in ps:
        p.grad = torch.ones_like(p)
    opt.step()
    other = adamw.AdamW([{"params": [torch.ones(5, device=device).requires_grad_(True)], "lr": 0.125}, {"params": [torch.ones(5, device=device).requires_grad_(True)]}])
    saved = other.state_dict()
    saved["param_groups"][1].update(options)
    before = [t.clone() for t in opt.moments()]
    with pytest.raises(ValueError):
        opt.load_state_dict(saved)
    assert opt.param_groups[0]["lr"] == 0.25 and opt.param_groups[1]["lr"] is rate and float(rate) == 0.5 and opt.param_groups[1]["eps"] == 1e-8
    assert all(torch.equal(a, b) for a, b in zip(before, opt.moments())) and int(opt.state[ps[0]]["step"]) == 1
    opt.step()


@pytest.mark.parametrize("device", DEVICES)
def test_a_programs_own_entries_of_the_groups(device):
    """What a schedule keeps beside the options is saved and loaded with them."""
    made = lambda: adamw.AdamW([torch.ones(5, device=device).requires_grad_(True)], lr=0.5)      # noqa: E731
    one, two = made(), made()
    one.param_groups[0].update(initial_lr=0.25, curve=torch.arange(3))
    two.load_state_dict(one.state_dict())
    assert two.param_groups[0]["initial_lr"] == 0.25 and two.param_groups[0]["curve"].tolist() == [0, 1, 2]
    two.load_state_dict(one.state_dict())
    two.step()


@pytest.mark.parametrize("device", DEVICES)
def test_a_loaded_learning_rate_of_another_form(device):
    """One number of another type or shape is that number."""
    rate = torch.tensor(0.5, device=device)
    for lr in (rate, 0.125):
        for saved_lr in (torch.tensor([0.25]), torch.tensor(0.25, dtype=torch.float64)):
            p = torch.zeros(5, device=device).requires_grad_(True)
            opt = adamw.AdamW([p], lr=lr)
            state = opt.state_dict()
            state["param_groups"][0]["lr"] = saved_lr
            opt.load_state_dict(state)
            p.grad = torch.ones_like(p)
            opt.step()
            assert torch.allclose(p.detach(), torch.full_like(p, -0.25), rtol=1e-6)
    assert float(rate) == 0.25


@pytest.mark.parametrize("device", DEVICES)
def test_a_refused_step_keeps_the_rates(device):
    """A step that is refused, for its rate or for a gradient, leaves the groups' rates too."""
    ps = [torch.ones(5, device=device).requires_grad_(True) for _ in range(2)]
    opt = adamw.AdamW([{"params": ps[:1], "lr": 0.25}, {"params": ps[1:], "lr": 0.5}])
    for p in ps:
        p.grad = torch.ones_like(p)
    calls = [lambda: opt.step(lr=-1.0)]
    if device == "cuda":
        calls.append(lambda: opt.step(lr=torch.tensor(0.1)))          # on the host

    def of_another_order():
        ps[1].grad = None
        ps[1].data = torch.ones(7, device=device)
        ps[1].grad = torch.ones(7, device=device)
        opt.step(lr=0.125)
    for call in (*calls, of_another_order):
        with pytest.raises(ValueError):
            call()
        assert [g["lr"] for g in opt.param_groups] == [0.25, 0.5] and int(opt.state[ps[0]]["step"]) == 0
    ps[1].data = torch.ones(5, device=device)
    ps[1].grad = None
    opt.step(lr=0.125)
    assert [g["lr"] for g in opt.param_groups] == [0.125, 0.125]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [8, 32])
def test_a_checkpoint_of_the_model_alone(bits, device, tmp_path):
    """Loaded weights are those that the next step starts from, also where the file holds no optimizer."""
    from torchmpi_b200.utils import checkpoint
    torch.manual_seed(0)
    a, b = (torch.nn.Linear(40, 30).to(BF).to(device) for _ in range(2))
    checkpoint.save(str(tmp_path / "model.pt"), a)
    opt = adamw.AdamW(b.parameters(), lr=1e-4, weight_decay=0.0, bits=bits)
    checkpoint.load(str(tmp_path / "model.pt"), b, opt)
    assert all(torch.equal(p, q) and torch.equal(opt.state[q]["master"], p.detach().float()) for p, q in zip(a.parameters(), b.parameters()))
    for p in b.parameters():
        p.grad = torch.ones_like(p)
    opt.step()
    for p, q in zip(a.parameters(), b.parameters()):          # a first step is as long as its rate
        want = p.detach().double() - 1e-4
        assert ((opt.state[q]["master"].double() - want).abs() <= 2.0 ** -20 * (want.abs() + 1e-4)).all()


@pytest.mark.parametrize("device", DEVICES)
def test_a_number_is_loaded_into_the_rate_on_the_device(device):
    """A captured step reads the tensor: a saved rate that is a number goes into it."""
    p = torch.zeros(5, device=device).requires_grad_(True)
    rate = torch.tensor(0.5, device=device)
    opt, other = adamw.AdamW([p], lr=rate), adamw.AdamW([torch.zeros(5, device=device).requires_grad_(True)], lr=0.25)
    p.grad = torch.ones_like(p)
    step = opt.step
    if device == "cuda":
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            opt.step()
        step = graph.replay
    opt.load_state_dict(other.state_dict())
    assert opt.param_groups[0]["lr"] is rate and float(rate) == 0.25
    step()
    assert torch.allclose(p.detach(), torch.full_like(p, -0.25), rtol=1e-6)
