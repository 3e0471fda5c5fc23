"""The gated delta rule (include/dcc_delta.h, dcc_hip.gated_delta_*, algos.algo_utils.fused.gated_delta) against the recurrence written
token by token in float64, its gradient against autograd of that recurrence and against differences.

Tolerances.  Keys have unit length, 0 <= beta <= 1 and g <= 0, so one token maps the state by a contraction: a rounding made at some
token is not amplified afterwards.  Per token an output collects at most about DK + 16 roundings of the products of its chunk and 4 of
the state update, each 2^-24 of the largest magnitude in play, and the updates of T tokens add up: fp32 results are held to
    2^-24 * (4 T + 2 DK + 64) * max|ref|          (gradients, a second recurrence over the first one's results: 4 times that),
16-bit results to half a step of their type on top (bf16 2^-8, fp16 2^-11 of the value)."""
import ctypes
import math
import itertools

import pytest
import torch

from algos.algo_utils import fused

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
NAMES = ("q", "k", "v", "g", "beta", "state")


def make(T, B, HK, H, DK, DV, dtype=torch.float32, reset=0.1, seed=0, device="cpu", beta=None):
    gen = torch.Generator().manual_seed(seed)
    n01 = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)
    unit = lambda x: x / x.norm(dim=-1, keepdim=True).clamp_min(1e-30)
    d = dict(q=unit(n01(T, B, HK, DK)), k=unit(n01(1, B, HK, DK) + 0.5 * n01(T, B, HK, DK)), v=n01(T, B, H, DV),
             g=-torch.nn.functional.softplus(n01(T, B, H) - 1.0), beta=torch.sigmoid(n01(T, B, H)), state=n01(B, H, DK, DV),
             masks=(torch.rand(T, B, generator=gen) >= reset).double())
    if beta is not None:
        d["beta"].fill_(beta)
    return {n: x.to(dtype if n in "qkv" else torch.float32).to(device) for n, x in d.items()}


def reference(d, scale, do=None, dstate=None, grads=False):
    """float64, token by token; {name: value} with the gradients of <do, o> + <dstate, last state> when asked."""
    x = {n: t.detach().double().cpu() for n, t in d.items() if t is not None}
    if grads:
        for n in NAMES:
            x[n].requires_grad_(True)
    q, k, v, g, beta, S, masks = (x.get(n) for n in NAMES + ("masks",))
    T, B, H, DV = v.shape
    rep = H // q.shape[2]
    outs = []
    for t in range(T):
        keep = torch.ones(B, dtype=torch.bool) if masks is None else masks[t] != 0
        S = torch.where(keep.view(B, 1, 1, 1), S * g[t].exp().view(B, H, 1, 1), torch.zeros((), dtype=torch.float64))
        kt, qt = k[t].repeat_interleave(rep, 1), q[t].repeat_interleave(rep, 1)
        u = beta[t].unsqueeze(-1) * (v[t] - torch.einsum("bhkv,bhk->bhv", S, kt))
        S = S + kt.unsqueeze(-1) * u.unsqueeze(-2)
        outs.append(scale * torch.einsum("bhkv,bhk->bhv", S, qt))
    o = torch.stack(outs) if outs else v.new_zeros(v.shape)
    r = dict(o=o.detach(), last=S.detach())
    if grads:
        got = torch.autograd.grad((o * do.double().cpu()).sum() + (S * dstate.double().cpu()).sum(), [x[n] for n in NAMES], allow_unused=True)
        r.update({"d" + n: (torch.zeros_like(x[n]) if gx is None else gx) for n, gx in zip(NAMES, got)})
    return r


def bound(T, DK, grad=False):
    return 2.0 ** -24 * (4 * T + 2 * DK + 64) * (4 if grad else 1)


def check(got, ref, T, DK, grad=False, what=""):
    ref = ref.to(torch.float64)
    g = got.detach().double().cpu()
    assert g.shape == ref.shape, what
    assert torch.isfinite(g).all(), what
    if ref.numel() == 0:
        return
    top = float(ref.abs().max())
    room = bound(T, DK, grad) * top + (HALF_STEP[got.dtype] * ref.abs() if got.dtype != torch.float32 else 0.0)
    if got.dtype == torch.float16:
        room = room + 2.0 ** -25          # half of the smallest float16 step
    worst = float(((g - ref).abs() - room).max())
    assert worst <= 0, "%s: %.3e over the bound (largest value %.3e)" % (what, worst, top)


# ---- CPU ---------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("T,B,HK,H,DK,DV", [(1, 1, 1, 1, 1, 1), (7, 3, 2, 4, 5, 6), (20, 2, 1, 3, 8, 4)])
def test_torch_form_is_the_recurrence(T, B, HK, H, DK, DV):
    d = make(T, B, HK, H, DK, DV)
    for n in NAMES:
        d[n].requires_grad_(True)
    do, ds = torch.randn(T, B, H, DV), torch.randn(B, H, DK, DV)
    o, S = fused.gated_delta(*[d[n] for n in NAMES], d["masks"])
    grads = torch.autograd.grad([o, S], [d[n] for n in NAMES], [do, ds])
    r = reference(d, DK ** -0.5, do, ds, grads=True)
    check(o, r["o"], T, DK, what="o")
    check(S, r["last"], T, DK, what="last")
    for n, x in zip(NAMES, grads):
        check(x, r["d" + n], T, DK, True, "d" + n)


def test_torch_form_gradient_against_differences():
    d = {n: t.double() for n, t in make(5, 2, 1, 2, 3, 2, reset=0.2, seed=3).items()}
    f = lambda *a: fused.gated_delta(*a, d["masks"], 0.7)
    assert torch.autograd.gradcheck(f, [d[n].requires_grad_(True) for n in NAMES], eps=1e-6, atol=1e-8)


def test_entry_points_validate_before_touching_the_device():
    import dcc_hip
    L = dcc_hip.load_library()
    buf = (ctypes.c_float * 64)()
    a = ctypes.addressof(buf)

    def seq(**kw):
        s = dcc_hip.DeltaSeq()
        s.T, s.B, s.HK, s.H, s.DK, s.DV, s.scale = 1, 1, 1, 1, 4, 4, 1.0
        s.q = s.k = s.v = s.g = s.beta = s.o = s.state0 = s.state1 = a
        for n, v in kw.items():
            setattr(s, n, v)
        return s

    for bad in (dict(DK=0), dict(DK=129), dict(DV=129), dict(DV=0), dict(HK=2, H=3), dict(H=0), dict(T=-1), dict(B=-1), dict(dtype=3),
                dict(q=None), dict(v=None), dict(beta=None), dict(o=None), dict(B=1 << 31), dict(T=(1 << 31) + 1)):
        s = seq(**bad)
        assert L.dcc_delta_fwd(ctypes.byref(s), None, None) == -1, bad
        assert b"dcc_delta_fwd" in L.dcc_last_error()
        assert L.dcc_delta_step(ctypes.byref(s), None) == -1, bad
    assert L.dcc_delta_fwd(None, None, None) == -1 and L.dcc_delta_step(None, None) == -1 and L.dcc_delta_bwd(None, None, None, None) == -1
    for bad in (dict(T=2), dict(T=0), dict(state0=None), dict(state1=None)):
        assert L.dcc_delta_step(ctypes.byref(seq(**bad)), None) == -1, bad
    g = dcc_hip.DeltaGrad()
    assert L.dcc_delta_bwd(ctypes.byref(seq()), ctypes.byref(g), None, None) == -1            # no checkpoint, no gradients
    g.ckpt = a
    assert L.dcc_delta_bwd(ctypes.byref(seq()), ctypes.byref(g), None, None) == -1
    g.dout = g.dq = g.dk = g.dv = g.dg = g.dbeta = a
    assert L.dcc_delta_bwd(ctypes.byref(seq(H=2)), ctypes.byref(g), None, None) == -1          # shared key heads need a workspace
    s = seq(B=0)
    assert L.dcc_delta_fwd(ctypes.byref(s), None, None) == 0 and L.dcc_delta_step(ctypes.byref(s), None) == 0
    assert L.dcc_delta_ckpt_floats(ctypes.byref(seq(T=17, B=2, H=3, HK=1))) >= 2 * 3 * 16
    assert L.dcc_delta_ckpt_floats(ctypes.byref(seq(DK=200))) == 0
    assert L.dcc_delta_bwd_workspace_floats(ctypes.byref(seq(T=10, B=2, H=3, HK=1))) >= 2 * 10 * 2 * 3 * 4


def test_no_cpu_path_behind_the_binding():
    import dcc_hip
    d = make(2, 1, 1, 1, 4, 4)
    with pytest.raises(dcc_hip.DccError):
        dcc_hip.gated_delta_fwd(*[d[n] for n in NAMES])
    with pytest.raises(dcc_hip.DccError):
        dcc_hip.gated_delta_step(*[d[n][0] for n in NAMES[:5]], d["state"])
    with pytest.raises(ValueError):
        fused.gated_delta(d["q"][0], d["k"][0], d["v"][0], d["g"], d["beta"])


# ---- GPU ---------------------------------------------------------------------------------------------------------------------------
SIZES = [(1, 1, 1, 1, 1, 1), (2, 3, 1, 1, 16, 16), (15, 2, 2, 2, 64, 64), (16, 5, 2, 4, 32, 48), (17, 3, 4, 4, 64, 64), (10, 70, 4, 4, 64, 64),
         (63, 2, 1, 3, 33, 17), (64, 2, 2, 2, 96, 80), (65, 1, 2, 2, 128, 128), (150, 4, 2, 2, 64, 64), (150, 2, 1, 5, 7, 100),
         (300, 1, 1, 2, 128, 40), (129, 2, 2, 2, 20, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_sequence_and_gradient(size, dtype):
    T, B, HK, H, DK, DV = size
    d = make(*size, dtype=dtype, reset=0.08, seed=T + DK, device="cuda")
    for n in NAMES:
        d[n].requires_grad_(True)
    gen = torch.Generator().manual_seed(9)
    do = torch.randn(T, B, H, DV, generator=gen).to(dtype).cuda()
    ds = torch.randn(B, H, DK, DV, generator=gen).cuda()
    o, S = fused.gated_delta(*[d[n] for n in NAMES], d["masks"])
    grads = torch.autograd.grad([o, S], [d[n] for n in NAMES], [do, ds])
    r = reference(d, DK ** -0.5, do, ds, grads=True)
    check(o, r["o"], T, DK, what="o")
    check(S, r["last"], T, DK, what="last")
    for n, x in zip(NAMES, grads):
        assert x.dtype == d[n].dtype and x.shape == d[n].shape
        check(x, r["d" + n], T, DK, True, "d" + n)


LONG = [(700, 1, 1, 2, 64, 64), (1000, 2, 2, 4, 33, 17), (1100, 1, 1, 1, 128, 128), (2100, 1, 1, 3, 16, 40), (1540, 2, 1, 2, 96, 20), (520, 3, 1, 1, 64, 96)]


@pytest.mark.gpu
@pytest.mark.parametrize("size", LONG, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype,reset", [(torch.float32, 0.0), (torch.float32, 0.01), (torch.bfloat16, 0.002)])
def test_long_sequences(size, dtype, reset):
    """few rows and many tokens: the segments that run side by side are joined to the sequence's own result and gradient"""
    T, B, HK, H, DK, DV = size
    d = make(*size, dtype=dtype, reset=reset, seed=T + DK, device="cuda")
    d["g"].mul_(0.05)                       # a long memory: states reach across segments
    for n in NAMES:
        d[n].requires_grad_(True)
    gen = torch.Generator().manual_seed(9)
    do = torch.randn(T, B, H, DV, generator=gen).to(dtype).cuda()
    ds = torch.randn(B, H, DK, DV, generator=gen).cuda()
    o, S = fused.gated_delta(*[d[n] for n in NAMES], d["masks"])
    grads = torch.autograd.grad([o, S], [d[n] for n in NAMES], [do, ds])
    r = reference(d, DK ** -0.5, do, ds, grads=True)
    check(o, r["o"], T, DK, what="o")
    check(S, r["last"], T, DK, what="last")
    for n, x in zip(NAMES, grads):
        check(x, r["d" + n], T, DK, True, "d" + n)


@pytest.mark.gpu
def test_a_restart_wipes_nan_across_segments():
    """1600 tokens of one row: a NaN at token 40, a restart at 700 -- everything from there on equals the clean run, as do its gradients"""
    size = T, B, HK, H, DK, DV = 1600, 1, 1, 2, 32, 32
    d = make(*size, reset=0.0, seed=13, device="cuda")
    d["masks"][700] = 0
    outs = []
    for dirty in (False, True):
        x = {n: t.clone() for n, t in d.items()}
        if dirty:
            x["v"][40] = float("nan")
        leaves = [x[n].requires_grad_(True) for n in NAMES]
        o, S = fused.gated_delta(*leaves, x["masks"])
        g = torch.autograd.grad([o[704:].sum() + S.sum()], leaves)
        outs.append([o[704:], S] + [y[704:] for y in g[:5]])
    for a, b in zip(*outs):
        assert torch.equal(a, b) and torch.isfinite(a).all()


@pytest.mark.gpu
@pytest.mark.parametrize("masked,state,dlast", list(itertools.product([False, True], repeat=3)))
def test_optional_operands(masked, state, dlast):
    import dcc_hip
    T, B, HK, H, DK, DV = size = (37, 3, 2, 2, 24, 40)
    d = make(*size, seed=5, device="cuda")
    if not masked:
        d["masks"] = None
    o, S, ck = dcc_hip.gated_delta_fwd(*[d[n] for n in NAMES[:5]], d["state"] if state else None, d["masks"], 0.3, want_ckpt=True)
    do = torch.randn(T, B, H, DV, device="cuda")
    ds = torch.randn(B, H, DK, DV, device="cuda") if dlast else None
    got = dcc_hip.gated_delta_bwd(*[d[n] for n in NAMES[:5]], d["masks"], 0.3, ck, do, ds)
    if not state:
        d["state"] = torch.zeros_like(d["state"])
    r = reference(d, 0.3, do, torch.zeros(B, H, DK, DV) if ds is None else ds, grads=True)
    check(o, r["o"], T, DK, what="o")
    check(S, r["last"], T, DK, what="last")
    for n, x in zip(NAMES, got):
        check(x, r["d" + n], T, DK, True, "d" + n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_operands_equal_contiguous_ones(dtype):
    """slices of one fused projection, batch-first tensors, expanded gates, offset (unaligned) views: same bits as contiguous copies"""
    T, B, HK, H, DK, DV = 35, 3, 2, 4, 24, 20
    d = make(T, B, HK, H, DK, DV, dtype=dtype, seed=11, device="cuda")
    s = dict(d)
    proj = torch.empty(B, T, 2 * HK * DK + H * DV + 3, dtype=dtype, device="cuda")
    a, b = HK * DK + 1, 2 * HK * DK + 1
    for n, lo, hi in (("q", 1, a), ("k", a, b), ("v", b, b + H * DV)):
        proj[..., lo:hi] = d[n].transpose(0, 1).reshape(B, T, -1)
        s[n] = proj[..., lo:hi].unflatten(-1, tuple(d[n].shape[2:])).transpose(0, 1)
        assert not s[n].is_contiguous() and torch.equal(s[n], d[n])
    s["g"] = torch.empty(H, B, T, device="cuda").copy_(d["g"].permute(2, 1, 0)).permute(2, 1, 0)
    d["beta"] = d["beta"][:, :, :1].expand(T, B, H).contiguous()
    s["beta"] = d["beta"][:, :, :1].expand(T, B, H)                      # stride 0 over the heads
    d["masks"] = d["masks"][:, :1].expand(T, B).contiguous()
    s["masks"] = d["masks"][:, :1].expand(T, B)
    outs = []
    for x in (d, s):
        leaves = [x[n].detach().requires_grad_(True) for n in NAMES]
        o, S = fused.gated_delta(*leaves, x["masks"])
        gen = torch.Generator(device="cuda").manual_seed(2)
        do = torch.randn(B, T, H, DV, generator=gen, device="cuda").to(dtype).transpose(0, 1)
        outs.append([o, S] + list(torch.autograd.grad([o, S], leaves, [do if x is s else do.contiguous(), torch.ones_like(S)])))
    for x, y in zip(*outs):
        assert torch.equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("low", [float("-inf"), torch.finfo(torch.float32).min, -1e30, -150.0])
def test_vanishing_decay_is_a_restart(low):
    """exp(g) == 0 in float32 equals a zero mask bit for bit, gradients of the neighbours included, and costs no digits around it"""
    size = T, B, HK, H, DK, DV = 40, 2, 2, 2, 32, 32
    d = make(*size, reset=0.0, seed=4, device="cuda")
    at = [0, 7, 8, 16, 31, 39]
    gl = d["g"].clone(); gl[at] = low
    m = torch.ones(T, B, device="cuda"); m[at] = 0
    outs = []
    for g, masks in ((gl, None), (d["g"], m)):
        leaves = [d["q"], d["k"], d["v"], g, d["beta"], d["state"]]
        leaves = [x.detach().clone().requires_grad_(True) for x in leaves]
        o, S = fused.gated_delta(*leaves, masks)
        outs.append([o, S] + list(torch.autograd.grad([o.sum() + S.sum()], leaves)))
    for x, y in zip(*outs):
        assert torch.equal(x, y) and torch.isfinite(x).all()
    assert (outs[0][5][at] == 0).all()              # dg at a restart
    assert (outs[0][7] == 0).all()                  # the first state is forgotten at t = 0
    r = reference(dict(d, masks=m), DK ** -0.5)
    check(outs[0][0], r["o"], T, DK, what="o")


@pytest.mark.gpu
def test_every_token_restarts_and_none_is_written():
    size = T, B, HK, H, DK, DV = 33, 2, 1, 2, 16, 16
    d = make(*size, reset=2.0, seed=6, device="cuda")       # all masks zero: o_t = scale beta (q.k) v
    o, S = fused.gated_delta(*[d[n] for n in NAMES], d["masks"], 1.0)
    qk = (d["q"].double() * d["k"].double()).sum(-1, keepdim=True)
    check(o, (d["beta"].double().unsqueeze(-1) * qk * d["v"].double()).cpu(), 1, DK, what="o")
    d = make(*size, reset=0.0, seed=6, device="cuda", beta=0.0)
    d["g"].zero_()                                          # nothing decays, nothing is written: the padding of a ragged batch
    o, S = fused.gated_delta(*[d[n] for n in NAMES], None)
    assert torch.equal(S, d["state"])
    leaves = [d[n].detach().requires_grad_(True) for n in NAMES]
    o, S = fused.gated_delta(*leaves, None)
    do = torch.randn_like(o)
    grads = torch.autograd.grad([o, S], leaves, [do, torch.ones_like(S)])
    r = reference(d | dict(masks=None), DK ** -0.5, do, torch.ones(S.shape), grads=True)
    for n, x in zip(NAMES, grads):
        check(x, r["d" + n], T, DK, True, "d" + n)


@pytest.mark.gpu
def test_equal_keys_and_full_writes_keep_their_digits():
    """identical unit keys with beta = 1: the chunk's triangular matrix is all ones, where a product form of its inverse cancels"""
    size = T, B, HK, H, DK, DV = 48, 2, 1, 1, 64, 32
    d = make(*size, reset=0.0, seed=8, device="cuda", beta=1.0)
    d["k"] = d["k"][:1].expand(T, B, HK, DK).contiguous()
    d["g"] = torch.full_like(d["g"], -1e-4)
    leaves = [d[n].detach().requires_grad_(True) for n in NAMES]
    o, S = fused.gated_delta(*leaves, None)
    do = torch.randn_like(o)
    grads = torch.autograd.grad([o, S], leaves, [do, torch.zeros_like(S)])
    r = reference(d | dict(masks=None), DK ** -0.5, do, torch.zeros(S.shape), grads=True)
    check(o, r["o"], T, DK, what="o")
    for n, x in zip(NAMES, grads):
        check(x, r["d" + n], T, DK, True, "d" + n)


@pytest.mark.gpu
def test_a_restart_wipes_nan_and_infinity():
    import dcc_hip
    size = T, B, HK, H, DK, DV = 40, 2, 1, 2, 32, 32
    d = make(*size, reset=0.0, seed=12, device="cuda")
    d["masks"][0] = 0
    d["masks"][32] = 0
    clean, S0 = fused.gated_delta(*[d[n] for n in NAMES], d["masks"])
    d["state"].fill_(float("nan"))
    dirty, S1 = fused.gated_delta(*[d[n] for n in NAMES], d["masks"])
    assert torch.equal(clean, dirty) and torch.equal(S0, S1)
    d["v"][3, 0, 0, 5] = float("inf")                        # row 0, head 0: its own row only, and only up to the restart at 32
    dirty, S1 = fused.gated_delta(*[d[n] for n in NAMES], d["masks"])
    assert torch.equal(clean[32:], dirty[32:]) and torch.equal(S0, S1)
    assert torch.equal(clean[:, 1], dirty[:, 1]) and torch.equal(clean[:, 0, 1], dirty[:, 0, 1])
    o, S = dcc_hip.gated_delta_step(*[d[n][0] for n in NAMES[:5]], d["state"], d["masks"][0])
    assert torch.isfinite(o).all() and torch.isfinite(S).all()


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(0, 3, 1, 2, 8, 8), (0, 0, 1, 1, 8, 8), (5, 0, 1, 1, 8, 8)])
def test_empty(size):
    T, B, HK, H, DK, DV = size
    d = make(*size, device="cuda")
    leaves = [d[n].detach().requires_grad_(True) for n in NAMES]
    o, S = fused.gated_delta(*leaves, d["masks"])
    assert o.shape == (T, B, H, DV) and torch.equal(S.detach(), d["state"])
    grads = torch.autograd.grad([o, S], leaves, [torch.ones_like(o), 2 * torch.ones_like(S)])
    assert torch.equal(grads[5], 2 * torch.ones_like(S))


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(1, 1, 1, 1, 1), (64, 4, 4, 64, 64), (5, 1, 3, 33, 17), (1000, 2, 6, 96, 80), (3, 2, 2, 128, 128), (700, 2, 4, 20, 64)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_one_token(size, dtype):
    import dcc_hip
    B, HK, H, DK, DV = size
    d = make(1, *size, dtype=dtype, reset=0.2, seed=B, device="cuda")
    r = reference(d, DK ** -0.5)
    args = [d[n][0] for n in NAMES[:5]]
    o, S = dcc_hip.gated_delta_step(*args, d["state"], d["masks"][0])
    check(o, r["o"][0], 1, DK, what="o")
    check(S, r["last"], 1, DK, what="state")
    inplace, out = d["state"].clone(), torch.empty_like(o)
    o2, S2 = dcc_hip.gated_delta_step(*args, inplace, d["masks"][0], None, out, inplace)
    assert S2 is inplace and o2 is out and torch.equal(o, o2) and torch.equal(S, S2)
    lead = torch.empty(B * H * DK * DV + 1, device="cuda")[1:].view(B, H, DK, DV).copy_(d["state"])      # a state 4 bytes off 16-byte alignment
    o3, S3 = dcc_hip.gated_delta_step(*args, lead, d["masks"][0])
    check(o3, r["o"][0], 1, DK, what="o unaligned")
    check(S3, r["last"], 1, DK, what="state unaligned")


@pytest.mark.gpu
def test_steps_continue_a_sequence():
    """prefill of 21 tokens, then 30 single tokens = one sequence of 51 (a run of the operators as a rollout uses them)"""
    import dcc_hip
    size = T, B, HK, H, DK, DV = 51, 6, 2, 4, 64, 48
    d = make(*size, reset=0.1, seed=21, device="cuda")
    r = reference(d, DK ** -0.5)
    o, S, _ = dcc_hip.gated_delta_fwd(*[d[n][:21] for n in NAMES[:5]], d["state"], d["masks"][:21])
    outs = [o]
    for t in range(21, T):
        o, S = dcc_hip.gated_delta_step(*[d[n][t] for n in NAMES[:5]], S, d["masks"][t], state_out=S)
        outs.append(o.unsqueeze(0))
    check(torch.cat(outs), r["o"], T, DK, what="o")
    check(S, r["last"], T, DK, what="last")


@pytest.mark.gpu
def test_same_bits_again_and_per_row():
    """no atomics: the same call gives the same bits; a row's results do not depend on the other rows of the batch"""
    size = T, B, HK, H, DK, DV = 100, 9, 2, 4, 64, 64
    d = make(*size, seed=30, device="cuda")

    def go(rows):
        leaves = [(d[n][rows] if n == "state" else d[n][:, rows]).detach().requires_grad_(True) for n in NAMES]
        o, S = fused.gated_delta(*leaves, d["masks"][:, rows])
        return [o, S] + list(torch.autograd.grad([o.square().sum() + S.square().sum()], leaves))
    a, b, c = go(slice(None)), go(slice(None)), go(slice(4, 5))
    for x, y, z in zip(a, b, c):
        assert torch.equal(x, y)
        assert torch.equal(x[4:5] if x.shape[0] == B else x[:, 4:5], z)


@pytest.mark.gpu
def test_other_stream_and_graph():
    """captured on another stream and replayed with new inputs, eager work between the replays: every replay equals the eager result"""
    import dcc_hip
    size = T, B, HK, H, DK, DV = 30, 4, 2, 4, 64, 64
    sets = [make(*size, seed=40 + i, device="cuda") for i in range(4)]
    buf = {n: x.clone() for n, x in sets[0].items()}
    do, ds = torch.randn(T, B, H, DV, device="cuda"), torch.randn(B, H, DK, DV, device="cuda")

    def work(d):
        o, S, ck = dcc_hip.gated_delta_fwd(*[d[n] for n in NAMES], d["masks"], want_ckpt=True)
        g = dcc_hip.gated_delta_bwd(*[d[n] for n in NAMES[:5]], d["masks"], None, ck, do, ds)
        o1, S1 = dcc_hip.gated_delta_step(*[d[n][0] for n in NAMES[:5]], S, d["masks"][0])
        return [o, S, o1, S1] + list(g)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        work(buf)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = work(buf)
    for i in (1, 2, 3, 1):
        for n in buf:
            buf[n].copy_(sets[i][n])
        graph.replay()
        got = [x.clone() for x in outs]
        torch.cuda.synchronize()
        for x, y in zip(got, work(sets[i])):
            assert torch.equal(x, y)


@pytest.mark.gpu
def test_binding_refuses():
    import dcc_hip
    d = make(4, 2, 2, 4, 8, 8, device="cuda")
    args = [d[n] for n in NAMES]
    ok = lambda a, m=None: dcc_hip.gated_delta_fwd(*a, m)
    ok(args, d["masks"])
    for i, bad in ((0, d["q"].double()), (0, d["q"][:3]), (0, d["q"].transpose(2, 3)), (1, d["k"].cpu()), (1, d["k"].bfloat16()),
                   (2, d["v"].double()), (2, d["v"][:, :, :3]), (2, d["v"][0]), (3, d["g"].double()), (3, d["g"][..., :2]), (4, d["beta"].half()),
                   (5, d["state"].transpose(2, 3)), (5, d["state"][:1]), (5, d["state"].double())):
        a = list(args)
        a[i] = bad
        with pytest.raises((ValueError, dcc_hip.DccError)):
            ok(a)
    with pytest.raises(ValueError):
        ok(args, d["masks"].bool())
    wide = make(2, 1, 1, 1, 129, 8, device="cuda")
    with pytest.raises(ValueError):
        ok([wide[n] for n in NAMES])
    o, S, ck = dcc_hip.gated_delta_fwd(*args, want_ckpt=True)
    with pytest.raises(ValueError):
        dcc_hip.gated_delta_bwd(*args[:5], None, None, ck[:-1], o)
    with pytest.raises(ValueError):
        dcc_hip.gated_delta_bwd(*args[:5], None, None, ck, o.bfloat16())
    one = [x[0] for x in args[:5]]
    with pytest.raises(ValueError):
        dcc_hip.gated_delta_step(*one, None)
    big = torch.zeros(2 * d["state"].numel(), device="cuda")
    n = d["state"].numel()
    with pytest.raises(ValueError):          # half over the state it reads
        dcc_hip.gated_delta_step(*one, big[:n].view_as(d["state"]), state_out=big[n // 2:n // 2 + n].view_as(d["state"]))
    with pytest.raises(ValueError):
        dcc_hip.gated_delta_step(*one, d["state"], state_out=torch.empty(3, device="cuda"))
    # results over operands
    flat = torch.zeros(4096, device="cuda")
    oshape, sshape = one[2].shape, d["state"].shape
    at = lambda start, shape: flat[start:start + math.prod(shape)].view(shape)
    v = at(0, oshape)
    for bad in (dict(out=v), dict(out=at(8, oshape)), dict(state_out=at(v.numel() - 1, sshape)),
                dict(out=at(1024, oshape), state_out=at(1024 + 4, sshape))):
        with pytest.raises(dcc_hip.DccError, match="apart"):
            dcc_hip.gated_delta_step(one[0], one[1], v, one[3], one[4], d["state"], **bad)
    with pytest.raises(dcc_hip.DccError, match="apart"):
        dcc_hip.gated_delta_step(*one, at(0, sshape), out=at(16, oshape))
    dcc_hip.gated_delta_step(one[0], one[1], v, one[3], one[4], d["state"], out=at(v.numel(), oshape), state_out=d["state"])
