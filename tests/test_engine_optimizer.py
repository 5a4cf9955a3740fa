"""The engine with an optimizer in the place of SGD: optimizers that were made earlier, and rates of the groups' own."""
import pytest
import torch

from mp_util import run_ranks
from torchmpi_b200.engine import AllReduceSGDEngine
from torchmpi_b200.ops import adamw


def _net(seed, dtype=torch.bfloat16):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Linear(20, 150), torch.nn.ReLU(), torch.nn.Linear(150, 10)).to(dtype)


def _data(seed, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return [{"input": torch.randn(16, 20, generator=g).to(dtype), "target": torch.randint(0, 10, (16,), generator=g)} for _ in range(4)]


class _Loss(torch.nn.Module):
    def forward(self, x, target):
        return torch.nn.functional.cross_entropy(x.float(), target)


def _states(opt):
    return [t.double().tolist() for p in opt.state for _, t in sorted(opt.state[p].items())]


def _made_earlier(rank, world, bits):
    """Every rank's optimizer has masters and averages of its own before the engine synchronises the parameters."""
    import torchmpi_b200 as mpi
    from torchmpi_b200 import nn as mpinn
    mpi.start(with_cuda=False)
    net = _net(rank)
    opt = adamw.AdamW(net.parameters(), lr=0.01, bits=bits)
    for s in _data(10 + rank)[: 2 + rank]:
        opt.zero_grad()
        _Loss()(net(s["input"]), s["target"]).backward()
        opt.step()
    opt.zero_grad()
    before = [p.detach().clone() for p in net.parameters()], _states(opt)
    engine = AllReduceSGDEngine(gradient_scale=1.0 / world, optimizer=lambda params: opt)
    started = {}
    engine.hooks["onStart"] = lambda state: started.update(weights=[p.detach().clone() for p in net.parameters()], states=_states(opt))
    engine.train(net, _Loss(), _data(3), lr=0.01, maxepoch=1)
    assert engine.own_optimizer is opt
    if rank == 0:                                        # rank 0's are everybody's, as they were
        assert all(torch.equal(a, b) for a, b in zip(started["weights"], before[0])) and started["states"] == before[1]
    mpinn.check_with_allreduce(net)
    out = [p.detach().float().reshape(-1).tolist() for p in net.parameters()], started["states"], _states(opt)
    mpi.stop()
    return out


@pytest.mark.parametrize("bits", [8, 32])
def test_an_optimizer_that_was_made_earlier(bits):
    got = run_ranks(_made_earlier, 2, bits, timeout=300)
    assert got[0] == got[1]


def _own_rates(rank, world):
    import torchmpi_b200 as mpi
    mpi.start(with_cuda=False)
    net, rate = _net(0), torch.tensor(0.01)
    before = [p.detach().clone() for p in net.parameters()]
    made = lambda ps: adamw.AdamW([{"params": ps[:2], "lr": 0.0, "weight_decay": 0.0}, {"params": ps[2:], "lr": rate}])      # noqa: E731
    engine = AllReduceSGDEngine(optimizer=made)
    engine.train(net, _Loss(), _data(3), lr=None, maxepoch=1)
    now = list(net.parameters())
    assert all(torch.equal(a, b) for a, b in zip(now[:2], before[:2])) and not any(torch.equal(a, b) for a, b in zip(now[2:], before[2:]))
    assert engine.own_optimizer.param_groups[0]["lr"] == 0.0 and engine.own_optimizer.param_groups[1]["lr"] is rate and float(rate) == torch.tensor(0.01).item()
    engine.train(net, _Loss(), _data(3), lr=0.02, maxepoch=1, maxsteps=1)
    assert [g["lr"] for g in engine.own_optimizer.param_groups] == [0.02, 0.02]
    # nothing else has rates of its own
    class Criterion(_Loss):
        def __init__(self):
            super().__init__()
            self.scale = torch.nn.Parameter(torch.ones(()))

        def forward(self, x, target):
            return super().forward(x * self.scale, target)
    before = [p.detach().clone() for p in net.parameters()]
    for call in (lambda: AllReduceSGDEngine().train(net, _Loss(), _data(3), lr=None, maxepoch=1), lambda: engine.train(net, Criterion(), _data(3), lr=None, maxepoch=1)):
        with pytest.raises(ValueError, match="lr"):
            call()
    assert all(torch.equal(a, b) for a, b in zip(net.parameters(), before))
    criterion = Criterion()
    engine.train(net, criterion, _data(3), lr=None, lrcriterion=0.1, maxepoch=1)
    assert float(criterion.scale) != 1.0
    mpi.stop()


def test_rates_of_the_optimizers_own_groups():
    run_ranks(_own_rates, 1, timeout=300)
