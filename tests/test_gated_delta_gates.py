"""Gradient of the gates of the gated delta rule over the whole range of decays, against the recurrence in float64.

dg_t = <dS'_t, S'_t> with S'_t = exp(g_t) S_{t-1} the state as token t finds it and dS'_t its gradient: a number of the size of exp(g_t).

Tolerance.  Every term that the kernel sums for dg_t has run through the decay of token t, and so have its roundings: relative to
    size_t = exp(g_t) |S_{t-1}|_F |dS'_t|_F
they are those of any other gradient (tests/test_gated_delta.py): 4 * 2^-24 * (4 T + 2 DK + 64).  A decay is exp of a float32 sum of at most
104 in size (below, it is a restart): its argument is off by up to 104 * 2^-24, and so is the decay relative to itself, once per factor that a
term holds; two of them at most.  That is 208 * 2^-24 more, less than the 256 * 2^-24 that the first bound has at its smallest."""
import math

import pytest
import torch

from algos.algo_utils import fused
from test_gated_delta import NAMES, bound, make


def gates_reference(d, scale, do, dstate):
    """dg [T,B,H] and size_t, by the recurrence and its reverse in float64"""
    q, k, v, g, beta, S, masks = (d[n].detach().double().cpu() for n in NAMES + ("masks",))
    do, dS = do.double().cpu() * scale, dstate.double().cpu()
    T, B, H, DV = v.shape
    rep = H // q.shape[2]
    wide = lambda x: x.repeat_interleave(rep, 1)
    before, us, al = [], [], []
    for t in range(T):
        a = torch.where(masks[t][:, None] != 0, g[t].exp(), torch.zeros((), dtype=torch.float64))
        Sd = S * a[..., None, None]
        u = beta[t].unsqueeze(-1) * (v[t] - (Sd * wide(k[t]).unsqueeze(-1)).sum(-2))
        S = Sd + wide(k[t]).unsqueeze(-1) * u.unsqueeze(-2)
        before.append(Sd); us.append(u); al.append(a)
    dg, size = torch.zeros_like(g), torch.zeros_like(g)
    for t in reversed(range(T)):
        kt, qt = wide(k[t]), wide(q[t])
        dS = dS + qt.unsqueeze(-1) * do[t].unsqueeze(-2)
        dr = beta[t].unsqueeze(-1) * (dS * kt.unsqueeze(-1)).sum(-2)
        dS = dS - kt.unsqueeze(-1) * dr.unsqueeze(-2)
        dg[t] = (dS * before[t]).sum((-1, -2))
        size[t] = dS.flatten(-2).norm(dim=-1) * before[t].flatten(-2).norm(dim=-1)
        dS = dS * al[t][..., None, None]
    return dg, size


def run(d, T, B, HK, H, DK, DV):
    gen = torch.Generator().manual_seed(1)
    do = torch.randn(T, B, H, DV, generator=gen).to(d["v"])
    ds = torch.randn(B, H, DK, DV, generator=gen).to(d["state"])
    leaves = [d[n].detach().requires_grad_(True) for n in NAMES]
    o, S = fused.gated_delta(*leaves, d["masks"])
    dg = torch.autograd.grad([o, S], leaves[3], [do, ds])[0]
    ref, size = gates_reference(d, DK ** -0.5, do, ds)
    over = (dg.double().cpu() - ref).abs() - bound(T, DK, True) * size
    assert float(over.max()) <= 0, "%.2e over; worst error relative to its size %.2e" % (
        float(over.max()), float(((dg.double().cpu() - ref).abs() / size.clamp_min(1e-300)).max()))


SIZES = [(16, 2, 2, 2, 64, 64), (40, 3, 1, 2, 32, 48), (33, 2, 2, 2, 128, 128), (700, 1, 1, 2, 64, 64)]


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("gate", [-0.1, -2.0, -5.0, -7.0, -10.0, -20.0, -40.0, -60.0])
def test_every_gate_alike(size, gate, dev):
    d = make(*size, reset=0.05, seed=5, device=dev)
    d["g"].fill_(gate)
    run(d, *size)


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_gates_of_all_sizes_side_by_side(size, dev):
    """from no decay at all to nearly a restart, token by token and head by head"""
    d = make(*size, reset=0.05, seed=6, device=dev)
    gen = torch.Generator().manual_seed(2)
    d["g"].copy_(-torch.exp(torch.empty(d["g"].shape).uniform_(math.log(1e-3), math.log(60.0), generator=gen)))
    run(d, *size)
