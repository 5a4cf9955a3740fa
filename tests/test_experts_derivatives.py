"""Derivatives of layers of experts and 8-bit checkpoints that are asked for in other ways than by one backward pass."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from torchmpi_b200.ops import act8, experts

gpu = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]
BF = torch.bfloat16


def _calls(device):
    """name -> (function of the tensors, the tensors)"""
    g = torch.Generator().manual_seed(0)
    new = lambda *s: torch.randn(s, generator=g).to(BF).to(device)
    logits = torch.randn(6, 4, generator=g).to(device)
    r = experts.route(logits, 2)
    off = torch.tensor([0, 2, 2, 5, 6], dtype=torch.int32, device=device)
    return {
        "grouped_linear": (lambda x, w, b: experts.grouped_linear(x, w, b, off), (new(6, 16), new(4, 24, 16), new(4, 24))),
        "grouped_linear with GELU": (lambda x, w, b: experts.grouped_linear(x, w, b, off, gelu=True), (new(6, 16), new(4, 24, 16), new(4, 24))),
        "route": (lambda l: experts.route(l, 2).weights, (logits,)),
        "route over all": (lambda l: experts.route(l, 2, renormalize=False).weights, (logits,)),
        "dispatch": (lambda x: experts.dispatch(x, r), (new(6, 16),)),
        "combine": (lambda rows, w: experts.combine(rows, r._replace(weights=w)), (new(12, 16), r.weights)),
        "experts.mlp": (lambda x, w, *p: experts.mlp(x, r._replace(weights=w), *p), (new(6, 16), r.weights, new(4, 24, 16), new(4, 24), new(4, 16, 24), new(4, 16))),
        "experts.mlp in 8 bits": (lambda x, w, *p: experts.mlp(x, r._replace(weights=w), *p, act8=True),
                                  (new(6, 16), r.weights, new(4, 24, 16), new(4, 24), new(4, 16, 24), new(4, 16))),
        "act8.mlp": (lambda *p: act8.mlp(*p), (new(6, 16), new(24, 16), new(24), new(16, 24), new(16))),
    }


NAMES = ("grouped_linear", "grouped_linear with GELU", "route", "route over all", "dispatch", "combine", "experts.mlp", "experts.mlp in 8 bits", "act8.mlp")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("name", NAMES)
def test_a_forward_tangent_is_refused_or_carried_on(name, graph, device):
    """An input with a forward-mode tangent, each in turn, with and without the grad mode: PyTorch's operations carry it on, the kernels' functions refuse it.  A
    result without a tangent would stand for a derivative of zero."""
    call, tensors = _calls(device)[name]
    for i, t in enumerate(tensors):
        with torch.set_grad_enabled(graph), fwd.dual_level():
            given = list(tensors)
            given[i] = fwd.make_dual(t, torch.ones_like(t))
            try:
                out = call(*given)
            except RuntimeError as e:
                assert "jvp" in str(e) and (device == "cuda" or "8" in name), e
            else:
                assert device == "cpu" and fwd.unpack_dual(out).tangent is not None, i


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("name", NAMES)
def test_without_a_tangent_results_are_the_same_inside_a_dual_level(name, device):
    call, tensors = _calls(device)[name]
    want = call(*tensors)
    with fwd.dual_level():
        assert torch.equal(call(*tensors), want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("E,k", [(4, 2), (5, 5), (40, 3), (200, 8)])
def test_the_gradient_of_a_token_with_a_nan(E, k, renormalize, device):
    """NaN at the logits that enter the token's weights (those of the chosen experts, or all), and nothing of it elsewhere, whoever computes it."""
    nan, inf = float("nan"), float("inf")
    g = torch.Generator().manual_seed(1)
    logits = torch.randn(9, E, generator=g)
    logits[1, 1] = nan                                     # one NaN among others
    logits[2] = nan                                        # nothing else
    logits[3], logits[3, 0], logits[3, 1] = -inf, 1.0, nan # fewer than k to choose, and a NaN
    logits[4], logits[4, 2] = -inf, nan                    # nothing to choose, and a NaN
    logits[5] = -inf                                       # padding
    logits[6, 3], logits[6, 0] = nan, -inf
    dw = torch.randn(9, k, generator=g)
    bad = torch.tensor([False, True, True, True, True, False, True, False, False])
    leaf = logits.to(device).requires_grad_(True)
    r = experts.route(leaf, k, renormalize)
    (got,) = torch.autograd.grad(r.weights, leaf, dw.to(device))
    got, weights, chosen = got.cpu(), r.weights.detach().cpu(), r.chosen.cpu().long()
    assert torch.equal(torch.isnan(weights), bad.unsqueeze(1).expand(9, k))
    mine = torch.zeros(9, E + 1, dtype=torch.bool).scatter_(1, torch.where(chosen >= 0, chosen, E), True)[:, :E]
    entered = mine if renormalize else torch.ones(9, E, dtype=torch.bool)
    assert torch.equal(torch.isnan(got), bad.unsqueeze(1) & entered)
    assert not got[bad][~torch.isnan(got[bad])].any() and not got[5].any()
    ordinary = logits[~bad].to(device).requires_grad_(True)          # the others are what they are without it
    (want,) = torch.autograd.grad(experts.route(ordinary, k, renormalize).weights, ordinary, dw[~bad].to(device))
    assert torch.equal(got[~bad], want.cpu())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("shape", [(1, 1), (5, 33), (4, 64), (2, 3, 40)], ids=str)
def test_the_gelu_gradient_is_linear_in_its_gradient(shape, dtype, device):
    """dz = dy gelu'(z): its derivative takes a gradient g to g gelu'(z), which is the function's own result for g; gelu(z) does not depend on dy."""
    g = torch.Generator().manual_seed(2)
    z, dy, gz = (torch.randn(shape, generator=g).to(dtype).to(device) for _ in range(3))
    a = act8.quantize(z)
    leaf = dy.clone().requires_grad_(True)
    dz, h = act8.gelu_gradient(leaf, a)
    want = act8.gelu_gradient(dy, a)
    assert dz.requires_grad and not h.requires_grad and torch.equal(dz, want[0]) and torch.equal(h, want[1])
    (got,) = torch.autograd.grad(dz, leaf, gz)
    assert got.dtype == dtype and torch.equal(got, act8.gelu_gradient(gz, a)[0])
    with torch.no_grad():
        assert not act8.gelu_gradient(leaf, a)[0].requires_grad
    for graph in (False, True):
        with torch.set_grad_enabled(graph), fwd.dual_level():
            dual = fwd.make_dual(dy, gz)
            if device == "cuda":
                with pytest.raises(RuntimeError, match="jvp"):
                    act8.gelu_gradient(dual, a)
            else:
                dz, h = act8.gelu_gradient(dual, a)
                assert torch.equal(fwd.unpack_dual(dz).tangent, act8.gelu_gradient(gz, a)[0]) and fwd.unpack_dual(h).tangent is None
    if device == "cuda":
        with pytest.raises(RuntimeError, match="once"):
            torch.autograd.grad(act8.gelu_gradient(leaf, a)[0], leaf, gz, create_graph=True)
