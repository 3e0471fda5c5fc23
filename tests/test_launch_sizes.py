"""Calls with more workgroups than one launch holds (2^32 threads): many small states in the gated delta rule, a list of very long matrices in
the orthogonalised updates.  Every element has its own closed form; 2^24 pairs of 256 threads are 2^32."""
import pytest
import torch

from test_gated_delta import bound

N = 2 ** 24 + 3


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [1, 3])
def test_many_pairs(heads):
    """[T, B, H, 1]: S = e^g S + k u and so on are products of numbers, written out in float64"""
    import dcc_hip
    T, H = 2, heads
    B = N // H + 1
    gen = torch.Generator(device="cuda").manual_seed(3)
    n01 = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    q, k, v = n01(T, B, H, 1).clamp(-2, 2), n01(T, B, H, 1).sign(), n01(T, B, H, 1)
    g, beta, S0 = -torch.rand(T, B, H, generator=gen, device="cuda"), torch.rand(T, B, H, generator=gen, device="cuda"), n01(B, H, 1, 1)
    m = (torch.rand(T, B, generator=gen, device="cuda") > 0.1).float()
    do, ds = n01(T, B, H, 1), n01(B, H, 1, 1)
    o, last, ck = dcc_hip.gated_delta_fwd(q, k, v, g, beta, S0, m, 1.0, want_ckpt=True)
    grads = dcc_hip.gated_delta_bwd(q, k, v, g, beta, m, 1.0, ck, do, ds)
    o1, S1 = dcc_hip.gated_delta_step(q[0], k[0], v[0], g[0], beta[0], S0, m[0], 1.0)
    Q, K, V, G, Be, S, M, DO, dS = (x.double().view(T, B, H) if x.dim() > 3 and x.shape[0] == T else x.double().view(B, H) if x.dim() > 3 else x.double()
                                    for x in (q, k, v, g, beta, S0, m, do, ds))
    Sd, U, R, al = [], [], [], []
    for t in range(T):
        a = G[t].exp() * M[t].unsqueeze(-1)
        sd = a * S
        r = V[t] - sd * K[t]
        S = sd + K[t] * Be[t] * r
        al.append(a); Sd.append(sd); R.append(r); U.append(Be[t] * r)
        got = o[t].view(B, H)
        assert float((got - S * Q[t]).abs().max()) <= bound(T, 1) * float((S * Q[t]).abs().max()), t
        if t == 0:
            assert float((o1.view(B, H) - S * Q[0]).abs().max()) <= bound(1, 1) * float((S * Q[0]).abs().max())
            assert float((S1.view(B, H) - S).abs().max()) <= bound(1, 1) * float(S.abs().max())
    assert float((last.view(B, H) - S).abs().max()) <= bound(T, 1) * float(S.abs().max())
    want = [[None] * T for _ in range(5)]
    for t in reversed(range(T)):
        dS = dS + Q[t] * DO[t]
        want[0][t] = (Sd[t] + K[t] * U[t]) * DO[t]
        du = dS * K[t]
        dr = Be[t] * du
        want[1][t], want[2][t], want[4][t] = dS * U[t] - Sd[t] * dr, dr, du * R[t]
        dS = dS - K[t] * dr
        want[3][t] = dS * Sd[t]
        dS = dS * al[t]
    for name, x, y in zip(("dq", "dk", "dv", "dg", "dbeta"), grads, want):
        for t in range(T):
            assert float((x[t].view(B, H) - y[t]).abs().max()) <= bound(T, 1, True) * float(y[t].abs().max()), (name, t)
    assert float((grads[5].view(B, H) - dS).abs().max()) <= bound(T, 1, True) * float(dS.abs().max())


@pytest.mark.gpu
def test_long_list():
    """20 rows of 2^25 + 1 numbers (5 million tiles in the last product): a row's one singular value is 1 after scaling, and p(1) = a + b + c"""
    import dcc_hip
    gen = torch.Generator(device="cuda").manual_seed(4)
    mats = [torch.randn(1, 2 ** 25 + 1, generator=gen, device="cuda") for _ in range(20)]
    got = dcc_hip.orthogonalize(mats)
    s = 1.0
    for _ in range(5):
        s = 3.4445 * s - 4.7750 * s ** 3 + 2.0315 * s ** 5
    for x, y in zip(mats, got):
        want = x.double() * (s / float(x.double().norm()))
        # the coefficients and the result in float32: 2^-24 each, through five steps of slope |p'(s)| < 9 at most near the fixed point's band
        assert float((y.double() - want).abs().max()) <= 2.0 ** -24 * 64 * float(want.abs().max())
