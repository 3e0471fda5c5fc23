"""Orthogonalised updates (include/dcc_ortho.h, dcc_hip.orthogonalize) against the Newton-Schulz steps in float64.

Tolerances, relative to the largest entry the result can have (singular values end below 1.3, so |x| <= 1.3 and |X|_F <= 1.3 sqrt(m)).
A product of depth K in float32 is off by at most K 2^-24 of the norms of its rows, but its roundings are independent: sqrt(K) 2^-24 is
taken, times 8.  Along a direction of small singular value a step multiplies an error by at most a = 3.4445 -- and by a^2 per step on
A = X X^T, for at most two steps before X X^T is formed anew (a^4 = 141); the polynomial itself has slope |b| + 2 |c| < 9 on [0, 1].  A
direction's error is thus at most 9 * 141 times a product's, in the Frobenius norm averaged over the directions, of which those that start
small enough to be amplified that far are few: the bound used is   |got - ref|_F <= 2^-24 * 8 sqrt(max(m, 16)) * 141 * |ref|_F / 8,
which for m = 256 is 1.3e-4; 16-bit results add half a step of their type."""
import ctypes
import math

import pytest
import torch

A, B, C = 3.4445, -4.7750, 2.0315
HALF_STEP = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def reference(G, steps=5, coeffs=(A, B, C), eps=1e-7):
    a, b, c = coeffs
    X = G.detach().double().cpu()
    tall = X.shape[-2] > X.shape[-1]
    X = X.mT if tall else X
    X = X / (X.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    for _ in range(steps):
        W = X @ X.mT
        X = a * X + b * (W @ X) + c * (W @ (W @ X))
    return X.mT if tall else X


def gradient_like(M, N, dtype=torch.float32, seed=0, noise=0.2):
    gen = torch.Generator().manual_seed(seed)
    r = max(1, min(M, N) // 4)
    G = (torch.randn(M, r, generator=gen) * torch.logspace(0, -2, r)) @ torch.randn(r, N, generator=gen) + noise * torch.randn(M, N, generator=gen)
    return (1e-3 * G).to(dtype)


def check(got, ref, what=""):
    m = max(16, min(ref.shape[-2:]))
    g = got.detach().double().cpu()
    assert g.shape == ref.shape and torch.isfinite(g).all(), what
    norm = float(ref.norm())
    tol = 2.0 ** -24 * math.sqrt(m) * 141 * norm + HALF_STEP[got.dtype] * norm
    off = float((g - ref).norm())
    assert off <= tol, "%s: off by %.3e, %.3e allowed (norm %.3e)" % (what, off, tol, norm)


# ---- CPU ---------------------------------------------------------------------------------------------------------------------------
def test_entry_points_validate_before_touching_the_device():
    import dcc_hip
    L = dcc_hip.load_library()
    buf = (ctypes.c_float * 4096)()
    a = (ctypes.addressof(buf) + 255) // 256 * 256
    one = lambda inp=a, out=a + 4096, M=4, N=4: (dcc_hip.OrthoMat * 1)(dcc_hip.OrthoMat(inp, out, M, N))
    go = lambda m, count=1, dt=0, steps=5, eps=1e-7, ws=a + 8192: L.dcc_orthogonalize(m, count, dt, steps, A, B, C, eps, ws, None)
    assert L.dcc_ortho_workspace_bytes(one(), 1, 0, 5) > 4 * 5 * 16
    assert go(None, 0) == 0 and go(one(M=0)) == 0 and go(one(inp=None, out=None, M=0)) == 0
    for bad in (dict(m=None), dict(m=one(), count=-1), dict(m=one(), dt=3), dict(m=one(), dt=-1), dict(m=one(), steps=0), dict(m=one(), steps=33),
                dict(m=one(), eps=-1.0), dict(m=one(), eps=float("nan")), dict(m=one(), ws=None), dict(m=one(), ws=a + 8196), dict(m=one(inp=None)),
                dict(m=one(out=None)), dict(m=one(M=-1)), dict(m=one(N=1 << 31)), dict(m=one(M=40000, N=40000)), dict(m=one(out=a)),
                dict(m=one(out=a + 32))):
        assert go(**bad) == -1, bad
        assert b"dcc_orthogonalize" in L.dcc_last_error()
    two = (dcc_hip.OrthoMat * 2)(dcc_hip.OrthoMat(a, a + 4096, 4, 4), dcc_hip.OrthoMat(a + 64, a + 4096, 4, 4))
    assert go(two, 2) == -1                                     # two results in one place
    far = [dcc_hip.OrthoMat(a + 64 * i, a + 4096 + 64 * i, 4, 4) for i in range(5)]
    far[3].out = a + 64 * 4 + 60                                # the last bytes of the last input
    assert go((dcc_hip.OrthoMat * 5)(*far), 5) == -1 and b"overlaps" in L.dcc_last_error()
    far[3].out, far[0].inp = a + 4096 + 64 * 9, a + 4096 + 64 * 9 - 4      # an input that ends inside an output
    assert go((dcc_hip.OrthoMat * 5)(*far), 5) == -1 and b"overlaps" in L.dcc_last_error()
    assert L.dcc_ortho_workspace_bytes(one(), 1, 0, 0) == 0


def test_no_cpu_path():
    import dcc_hip
    with pytest.raises(dcc_hip.DccError):
        dcc_hip.orthogonalize(torch.ones(4, 4))
    assert dcc_hip.orthogonalize([]) == []


# ---- GPU ---------------------------------------------------------------------------------------------------------------------------
SHAPES = [(1, 1), (1, 300), (300, 1), (2, 2), (16, 16), (31, 33), (64, 64), (65, 64), (63, 130), (96, 500), (500, 96), (128, 128), (127, 129), (200, 299),
          (200, 301), (256, 440), (256, 2704), (2704, 256), (257, 1031), (40, 9001), (9001, 40), (640, 700)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "%dx%d" % s)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_matrix(shape, dtype):
    import dcc_hip
    G = gradient_like(*shape, dtype=dtype, seed=shape[0]).cuda()
    before = G.clone()
    X = dcc_hip.orthogonalize(G)
    assert X.dtype == dtype and torch.equal(G, before)
    check(X, reference(G), "%dx%d" % shape)


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [1, 2, 3, 4, 6, 7])
@pytest.mark.parametrize("shape", [(48, 64), (48, 300), (300, 48)])
def test_steps(steps, shape):
    import dcc_hip
    G = gradient_like(*shape, seed=steps).cuda()
    check(dcc_hip.orthogonalize(G, steps=steps), reference(G, steps))
    check(dcc_hip.orthogonalize(G, steps=steps, coeffs=(1.875, -1.25, 0.375)), reference(G, steps, (1.875, -1.25, 0.375)))


# large and nearly square (step by step), and long (many tiles of X <- Q X): rows of a multiple of four or not, either way round
@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(705, 705), (720, 901), (1030, 772), (200, 16388), (200, 16389), (16388, 200), (16389, 201)], ids=lambda s: "%dx%d" % s)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_large(shape, dtype):
    import dcc_hip
    G = gradient_like(*shape, dtype=dtype, seed=shape[1]).cuda()
    check(dcc_hip.orthogonalize(G), reference(G), "%dx%d" % shape)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(720, 901), (200, 16388), (16389, 201)], ids=lambda s: "%dx%d" % s)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_in_two_groups_and_off_alignment(shape, dtype):
    """six steps (X X^T is formed twice on the m x m side), from and to places that are aligned to one element only"""
    import dcc_hip
    G = gradient_like(*shape, dtype=dtype, seed=7)
    n = G.numel()
    src, dst = torch.zeros(n + 1, dtype=dtype, device="cuda"), torch.zeros(n + 2, dtype=dtype, device="cuda")
    src[1:].copy_(G.reshape(-1))
    X, out = src[1:].view(shape), dst[1:-1].view(shape)
    dcc_hip.orthogonalize(X, steps=6, out=out)
    check(out, reference(G, 6), "%dx%d" % shape)
    assert float(dst[0]) == 0.0 and float(dst[-1]) == 0.0


@pytest.mark.gpu
def test_list_equals_single_calls():
    """a list of 45 matrices of all kinds (more than one launch holds) gives the bits of 45 lists of one of the same tile width"""
    import dcc_hip
    gen = torch.Generator().manual_seed(3)
    shapes = [(int(torch.randint(1, 200, (1,), generator=gen)), int(torch.randint(1, 400, (1,), generator=gen))) for _ in range(45)]
    mats = [gradient_like(m, n, seed=i).cuda() for i, (m, n) in enumerate(shapes)]
    outs = [torch.empty_like(x) for x in mats]
    got = dcc_hip.orthogonalize(mats, out=outs)
    assert all(a is b for a, b in zip(got, outs))
    for x, y in zip(mats, got):
        assert torch.equal(dcc_hip.orthogonalize(x), y)
        check(y, reference(x), str(tuple(x.shape)))
    batch = torch.stack([gradient_like(20, 30, seed=i) for i in range(6)]).view(2, 3, 20, 30).cuda()
    check(dcc_hip.orthogonalize(batch).view(6, 20, 30), reference(batch.view(6, 20, 30)))
    assert dcc_hip.orthogonalize(torch.empty(0, 5, 7, device="cuda")).shape == (0, 5, 7)
    assert dcc_hip.orthogonalize([torch.empty(0, 7, device="cuda"), mats[0]])[0].shape == (0, 7)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(37, 50), (50, 200)])
def test_scale_of_the_gradient(shape):
    """sums of squares that leave float32 in either direction; zero stays zero; a NaN reaches its own matrix only"""
    import dcc_hip
    G = gradient_like(*shape).cuda()
    for s in (1e-30, 1e30, 1.0):
        check(dcc_hip.orthogonalize(G * s, eps=0.0), reference(G * s, eps=0.0), "scale %g" % s)
    check(dcc_hip.orthogonalize(G * 1e-5, eps=1e-3), reference(G * 1e-5, eps=1e-3))
    Z = torch.zeros_like(G)
    bad = G.clone()
    bad[0, 0] = float("nan")
    z, x, y = dcc_hip.orthogonalize([Z, bad, G])
    assert torch.equal(z, Z) and torch.isnan(x).any()
    check(y, reference(G))


@pytest.mark.gpu
def test_rank_one_and_orthogonal_inputs():
    import dcc_hip
    u, v = torch.randn(70, 1, generator=torch.Generator().manual_seed(1)), torch.randn(1, 90, generator=torch.Generator().manual_seed(2))
    G = (u @ v).cuda()
    # the other directions hold the input's own rounding, which the steps amplify by a^5 = 485: compared through the strong one
    X = dcc_hip.orthogonalize(G).double().cpu()
    R = reference(G)
    un, vn = u.double() / u.double().norm(), v.double() / v.double().norm()
    assert abs(float(un.T @ (X - R) @ vn.T)) <= 2.0 ** -24 * 8 * math.sqrt(90) * 9
    Q = torch.linalg.qr(torch.randn(64, 64, generator=torch.Generator().manual_seed(4)))[0].contiguous().cuda()
    check(dcc_hip.orthogonalize(Q), reference(Q))


@pytest.mark.gpu
def test_other_stream_and_graph():
    import dcc_hip
    shapes = [(64, 300), (300, 64), (128, 128), (33, 2000)]
    sets = [[gradient_like(m, n, seed=10 * i + j).cuda() for j, (m, n) in enumerate(shapes)] for i in range(4)]
    buf = [x.clone() for x in sets[0]]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        eager = dcc_hip.orthogonalize(buf)
    torch.cuda.synchronize()
    for x, y in zip(eager, dcc_hip.orthogonalize(sets[0])):
        assert torch.equal(x, y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = dcc_hip.orthogonalize(buf)
    for i in (1, 2, 3, 1):
        for x, y in zip(buf, sets[i]):
            x.copy_(y)
        graph.replay()
        got = [x.clone() for x in outs]
        torch.cuda.synchronize()
        for x, y in zip(got, dcc_hip.orthogonalize(sets[i])):
            assert torch.equal(x, y)


@pytest.mark.gpu
def test_binding_refuses():
    import dcc_hip
    G = torch.randn(8, 12, device="cuda")
    for bad in (G.t(), G[0], G.double(), [G, G.bfloat16()], [G, G.cpu()], G.int()):
        with pytest.raises((ValueError, dcc_hip.DccError)):
            dcc_hip.orthogonalize(bad)
    for kw in (dict(out=G), dict(out=torch.empty(12, 8, device="cuda")), dict(out=torch.empty(8, 12, device="cuda", dtype=torch.bfloat16)),
               dict(steps=0), dict(steps=33), dict(coeffs=(1.0, 2.0)), dict(eps=-1.0)):
        with pytest.raises((ValueError, dcc_hip.DccError)):
            dcc_hip.orthogonalize(G, **kw)
    with pytest.raises(ValueError):
        dcc_hip.orthogonalize([G, G], out=[torch.empty_like(G)])
