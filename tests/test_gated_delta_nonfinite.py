"""Infinities and NaN in a sequence of the gated delta rule reach what the recurrence, taken token by token, lets them reach, in the results
and in the gradients; a restart ends them wherever it lies.

The reference is the recurrence and its reverse in float64, with restarts selected.  What is finite there has to be finite and within the
bound of tests/test_gated_delta.py (relative to the largest finite entry); what is not finite there must not be finite."""
import pytest
import torch

from algos.algo_utils import fused
from test_gated_delta import HALF_STEP, NAMES, bound, make

OUTS = ("o", "last") + tuple("d" + n for n in NAMES)


def reference(d, scale, do, dstate):
    q, k, v, g, beta, S, masks = (d[n].detach().double().cpu() for n in NAMES + ("masks",))
    do, dS = do.double().cpu() * scale, dstate.double().cpu()
    T, B, H, DV = v.shape
    HK, DK = q.shape[2:]
    rep = H // HK
    wide = lambda x: x.repeat_interleave(rep, 1)
    fold = lambda x: x.view(B, HK, rep, DK).sum(2)
    before, us, rs, outs = [], [], [], []
    cut = lambda t: ((masks[t] == 0)[:, None] | (g[t] < -104.0))[..., None, None]
    zero = torch.zeros((), dtype=torch.float64)
    for t in range(T):
        Sd = torch.where(cut(t), zero, S * g[t].exp()[..., None, None])
        r = v[t] - (Sd * wide(k[t]).unsqueeze(-1)).sum(-2)
        u = beta[t].unsqueeze(-1) * r
        S = Sd + wide(k[t]).unsqueeze(-1) * u.unsqueeze(-2)
        outs.append(scale * (S * wide(q[t]).unsqueeze(-1)).sum(-2))
        before.append(Sd); us.append(u); rs.append(r)
    res = dict(o=torch.stack(outs), last=S, dq=torch.zeros_like(q), dk=torch.zeros_like(k), dv=torch.zeros_like(v), dg=torch.zeros_like(g),
               dbeta=torch.zeros_like(beta))
    for t in reversed(range(T)):
        kt, qt = wide(k[t]).unsqueeze(-1), wide(q[t]).unsqueeze(-1)
        dS = dS + qt * do[t].unsqueeze(-2)
        res["dq"][t] = fold(((before[t] + kt * us[t].unsqueeze(-2)) * do[t].unsqueeze(-2)).sum(-1))
        du = (dS * kt).sum(-2)
        dr = beta[t].unsqueeze(-1) * du
        res["dbeta"][t], res["dv"][t] = (du * rs[t]).sum(-1), dr
        res["dk"][t] = fold((dS * us[t].unsqueeze(-2)).sum(-1) - (before[t] * dr.unsqueeze(-2)).sum(-1))
        dS = dS - kt * dr.unsqueeze(-2)
        c = cut(t)
        res["dg"][t] = torch.where(c[..., 0, 0], zero, (dS * before[t]).sum((-1, -2)))
        dS = torch.where(c, zero, dS * g[t].exp()[..., None, None])
    res["dstate"] = dS
    return res


def compare(d, size, dirty_do=None):
    T, B, HK, H, DK, DV = size
    gen = torch.Generator().manual_seed(1)
    do = torch.randn(T, B, H, DV, generator=gen).to(d["v"])
    ds = torch.randn(B, H, DK, DV, generator=gen).to(d["state"])
    if dirty_do:
        dirty_do(do, ds)
    leaves = [d[n].detach().requires_grad_(True) for n in NAMES]
    o, S = fused.gated_delta(*leaves, d["masks"])
    got = [o, S] + list(torch.autograd.grad([o, S], leaves, [do, ds]))
    ref = reference(d, DK ** -0.5, do, ds)
    for n, x in zip(OUTS, got):
        r, y = ref[n], x.detach().double().cpu()
        fin = torch.isfinite(r)
        assert torch.equal(torch.isfinite(y), fin), "%s: %d places finite, %d should be" % (n, int(torch.isfinite(y).sum()), int(fin.sum()))
        if fin.any():
            y, r = y[fin], r[fin]
            room = bound(T, DK, n[0] == "d") * float(r.abs().max()) + (HALF_STEP[x.dtype] * r.abs() if x.dtype != torch.float32 else 0.0)
            assert float(((y - r).abs() - room).max()) <= 0, n
    return ref


SIZES = [(48, 2, 2, 2, 16, 16), (40, 2, 1, 2, 64, 48), (31, 1, 1, 1, 128, 128), (37, 2, 2, 2, 33, 17), (35, 1, 1, 2, 128, 20), (700, 1, 1, 2, 32, 40)]
NAN, INF = float("nan"), float("inf")
# operand, value, token that holds it (of its first row and head), tokens that restart
PLACES = [("v", NAN, 5, (9,)), ("v", INF, 5, (6,)), ("v", -INF, 3, ()), ("v", NAN, 17, (20, 30)), ("k", NAN, 7, (8, 12)), ("k", INF, 0, (2,)),
          ("q", NAN, 6, ()), ("q", INF, 18, (19,)), ("beta", NAN, 4, (11,)), ("beta", INF, 15, (16,)), ("g", NAN, 3, (5,)), ("g", NAN, 5, (5,)),
          ("g", INF, 2, (13,)), ("state", NAN, None, (5,)), ("state", INF, None, (17,)), ("state", NAN, None, ()), ("do", NAN, 9, (4, 12)),
          ("do", INF, 19, (2, 18)), ("dstate", NAN, None, (7,)), ("dstate", -INF, None, (2, 19)), ("v", NAN, 15, (16,)), ("k", NAN, 16, (17,))]


def place(size, what, value, at, restarts, device, dtype=torch.float32):
    T, B, HK, H, DK, DV = size
    d = make(*size, dtype=dtype, reset=0.0, seed=T + DK, device=device)
    for t in restarts:
        d["masks"][t, 0] = 0
    spoil = None
    if what in ("do", "dstate"):
        def spoil(do, ds):
            if what == "do":
                do[at, 0, 0, DV // 2] = value
            else:
                ds[0, 0, DK // 2, DV - 1] = value
    elif what == "state":
        d["state"][0, 0, DK - 1, DV // 2] = value
    elif what in ("g", "beta"):
        d[what][at, 0, 0] = value
    else:
        d[what][at, 0, 0, -1] = value
    return d, spoil


@pytest.mark.gpu
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("what,value,at,restarts", PLACES)
def test_reach(size, what, value, at, restarts):
    d, spoil = place(size, what, value, at, restarts, "cuda")
    compare(d, size, spoil)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("what,value,at,restarts", PLACES[:8])
def test_reach_of_16_bit_operands(dtype, what, value, at, restarts):
    size = (40, 2, 1, 2, 64, 48)
    d, spoil = place(size, what, value, at, restarts, "cuda", dtype)
    compare(d, size, spoil)


@pytest.mark.gpu
def test_reach_across_segments():
    """few rows, many tokens: in one segment a NaN without a restart behind it, in another with one, a state that is not finite"""
    size = (1600, 1, 1, 2, 32, 32)
    for spots in ([("v", 40, 0), ("masks", 700, 0)], [("k", 703, 0), ("masks", 705, 0), ("v", 1200, 1)], [("state", 0, 0), ("masks", 300, 0)],
                  [("beta", 900, 1), ("masks", 899, 0), ("masks", 901, 0)]):
        d = make(*size, reset=0.0, seed=3, device="cuda")
        d["g"].mul_(0.05)
        for n, t, h in spots:
            if n == "masks":
                d[n][t] = 0
            elif n == "state":
                d[n][0, h] = NAN
            elif n == "beta":
                d[n][t, 0, h] = INF
            else:
                d[n][t, 0, 0 if n == "k" else h, 3] = NAN
        compare(d, size)


@pytest.mark.gpu
def test_sequence_and_steps_agree_on_what_is_finite():
    """a rollout's steps and the update's sequence of the same tokens (garbage behind the end of an episode, then a restart in mid-chunk)"""
    import dcc_hip
    size = T, B, HK, H, DK, DV = 40, 4, 2, 2, 32, 32
    d = make(*size, reset=0.0, seed=9, device="cuda")
    d["masks"][11, 1], d["masks"][27, 2], d["masks"][30, 3] = 0, 0, 0
    d["v"][10, 1], d["k"][26, 2], d["g"][29, 3] = NAN, INF, NAN
    o, last = fused.gated_delta(*[d[n] for n in NAMES], d["masks"])
    S, outs = d["state"].clone(), []
    for t in range(T):
        x, S = dcc_hip.gated_delta_step(*[d[n][t] for n in NAMES[:5]], S, d["masks"][t], state_out=S)
        outs.append(x)
    outs = torch.stack(outs)
    assert torch.equal(torch.isfinite(o), torch.isfinite(outs)) and torch.equal(torch.isfinite(last), torch.isfinite(S))
    assert torch.isfinite(o[11:, 1]).all() and torch.isfinite(o[:10, 1]).all() and torch.isfinite(last[1]).all()
    fin = torch.isfinite(outs)
    assert float((o[fin] - outs[fin]).abs().max()) <= 2 * bound(T, DK) * float(outs[fin].abs().max())


def test_the_reference_itself():
    """the reversed recurrence is the gradient of the plain one (finite inputs), and a restart ends a NaN in it"""
    size = (12, 2, 1, 2, 5, 4)
    d = {n: x.double() for n, x in make(*size, seed=2).items()}
    gen = torch.Generator().manual_seed(1)
    do, ds = torch.randn(12, 2, 2, 4, generator=gen).double(), torch.randn(2, 2, 5, 4, generator=gen).double()
    leaves = [d[n].requires_grad_(True) for n in NAMES]
    o, S = fused.gated_delta(*leaves, d["masks"])
    ref = reference(d, 5 ** -0.5, do, ds)
    for n, x in zip(OUTS, [o, S] + list(torch.autograd.grad([o, S], leaves, [do, ds]))):
        assert torch.allclose(x, ref[n], rtol=1e-12, atol=1e-12), n
    d, _ = place(size, "v", NAN, 3, (7,), "cpu")
    ref = reference(d, 1.0, do, ds)
    assert torch.isnan(ref["o"][3:7, 0, 0]).any() and torch.isfinite(ref["o"][7:]).all() and torch.isfinite(ref["o"][:3]).all()
    assert torch.isfinite(ref["dv"]).all() and torch.isfinite(ref["dq"][:3]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(1100, 1, 1, 3, 32, 40), (1300, 1, 2, 2, 80, 7), (790, 2, 1, 1, 128, 128)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("what,at,restarts", [("v", 3, ()), ("state", None, ()), ("k", 500, ()), ("v", 40, (700,)), ("do", -3, ()), ("dstate", None, ()),
                                              ("do", -300, (200,))])
def test_a_long_decay_is_no_restart(size, what, at, restarts):
    """few rows, many tokens, decays whose product over a segment is 0 in float32: what is not finite stays until a restart, as token by token"""
    if at is not None and at < 0:
        at += size[0]
    d, spoil = place(size, what, NAN, at, restarts, "cuda")
    d["g"].fill_(-0.7)              # exp(-0.7 * 256) is 0
    ref = compare(d, size, spoil)
    if not restarts:
        assert not torch.isfinite(ref["last" if what in ("v", "state", "k") else "dstate"][0, 0]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(40, 3, 1, 2, 32, 48), (1100, 1, 1, 2, 64, 20)], ids=lambda s: "x".join(map(str, s)))
def test_finite_and_not_in_turn_in_a_graph(size):
    """replays on inputs with and without such values equal the eager calls: nothing of the one is left for the other"""
    import dcc_hip
    T, B, HK, H, DK, DV = size
    sets = [make(*size, reset=0.05, seed=50 + i, device="cuda") for i in range(4)]
    sets[1]["v"][T // 2, 0, 1, 3], sets[2]["k"][5, 0, 0, 1], sets[2]["state"][0, 1, 2, 2] = NAN, INF, NAN
    do, ds = torch.randn(T, B, H, DV, device="cuda"), torch.randn(B, H, DK, DV, device="cuda")
    buf = {n: x.clone() for n, x in sets[0].items()}

    def work(d):
        o, S, ck = dcc_hip.gated_delta_fwd(*[d[n] for n in NAMES], d["masks"], want_ckpt=True)
        return [o, S] + list(dcc_hip.gated_delta_bwd(*[d[n] for n in NAMES[:5]], d["masks"], None, ck, do, ds))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        work(buf)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = work(buf)
    for i in (1, 3, 2, 0, 1):
        for n in buf:
            buf[n].copy_(sets[i][n])
        graph.replay()
        got = [x.clone() for x in outs]
        torch.cuda.synchronize()
        for x, y in zip(got, work(sets[i])):
            assert torch.equal(torch.nan_to_num(x, 7e30), torch.nan_to_num(y, 7e30))
