"""What the flat optimizers do with the state of another optimizer, or of other parameters: refuse it, and keep what they hold."""
import pytest
import torch

from algos.algo_utils.optim import FlatAdam, FlatMuon

SHAPES = [(16, 16), (256,), (3, 20), (20, 17)]


def params(shapes=SHAPES, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(*s, generator=gen)) for s in shapes]


def stepped(cls, shapes=SHAPES, seed=0, **kw):
    ps = params(shapes, seed)
    opt = cls(ps, lr=1e-2, **kw)
    gen = torch.Generator().manual_seed(seed + 1)
    for p in ps:
        p.grad = torch.randn(p.shape, generator=gen) if p.grad is None else p.grad.add_(torch.randn(p.shape, generator=gen))
    opt.step()
    return opt


def held(opt):
    return [opt.exp_avg.clone(), opt.exp_avg_sq.clone(), torch.tensor(opt.step_count), torch.tensor(opt.param_groups[0]["lr"])]


@pytest.mark.parametrize("shapes", [SHAPES, [(16, 16), (256,)], [(32, 32), (4, 256), (64, 16)], [(16, 16)]])
def test_muon_refuses_the_state_of_adam(shapes):
    """also where every count of elements fits: the moments belong to other parameters, or are not a momentum"""
    opt = stepped(FlatMuon, shapes)
    before = held(opt)
    for sd in (stepped(torch.optim.Adam, shapes, 5).state_dict(), stepped(FlatAdam, shapes, 5).state_dict()):
        with pytest.raises(ValueError, match="another optimizer"):
            opt.load_state_dict(sd)
        assert all(torch.equal(x, y) for x, y in zip(before, held(opt)))


def test_adam_checks_every_shape_before_it_touches_its_moments():
    opt = stepped(FlatAdam)
    before = held(opt)
    good = stepped(torch.optim.Adam, seed=7).state_dict()
    wrong = stepped(torch.optim.Adam, SHAPES[:3] + [(17, 20)], 7).state_dict()          # the last one turned: the same count of elements
    short = stepped(torch.optim.Adam, SHAPES[:3], 7).state_dict()
    other = stepped(torch.optim.Adam, SHAPES[:3] + [(5, 5)], 7).state_dict()
    for sd in (wrong, short, other):
        with pytest.raises(ValueError, match="parameter"):
            opt.load_state_dict(sd)
        assert all(torch.equal(x, y) for x, y in zip(before, held(opt)))
    opt.load_state_dict(good)
    for i, (off, s) in enumerate(zip(opt._offsets, SHAPES)):
        n = torch.Size(s).numel()
        assert torch.equal(opt.exp_avg[off:off + n].view(s), good["state"][i]["exp_avg"])
        assert torch.equal(opt.exp_avg_sq[off:off + n].view(s), good["state"][i]["exp_avg_sq"])


@pytest.mark.parametrize("cls", [FlatAdam, FlatMuon])
def test_own_state_of_other_parameters(cls):
    opt = stepped(cls)
    before = held(opt)
    with pytest.raises(ValueError, match="layout"):
        opt.load_state_dict(stepped(cls, [(16, 16), (256,), (3, 20), (21, 17)]).state_dict())
    assert all(torch.equal(x, y) for x, y in zip(before, held(opt)))
    twin = stepped(cls, seed=9)
    opt.load_state_dict(twin.state_dict())
    assert all(torch.equal(x, y) for x, y in zip(held(twin), held(opt)))
