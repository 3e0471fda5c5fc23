"""Accuracy of the orthogonalised updates (dcc_hip.orthogonalize), path by path, in bounds close enough to see one part of a product missing.

m x m side (float64; m <= 704, or n long against m), at most five steps: roundings of 2^-53 grow by at most a^2 = 12 per step of A, four times
before the last, and enter with |b| and sums of m terms: below 1e-9 of the result for every shape here.  What is left is the one rounding
of the result.  So the distance from the exact result is that of the exact result from its own rounding, and 1e-9:
    |got - ref| <= |round(ref) - ref| (1 + 4 / sqrt(N)) + 1e-9 |ref|         (N entries: how far two such sums differ by chance)

Step by step (large and nearly square): products of 24 bits (float32, float16), or of 16 bits beside a float32 X (bfloat16), summed in
float32.  The sum of a product of depth K has K / 32 roundings, of partial sums that grow with it: c = 1 + sqrt(K / 96) of them in all, 2^-24
each, of |X|_2 |X|_F at most, as does the rounding of the parts.  An error of A enters X with |b| = 4.775; an error of X grows by at most a =
3.4445 a step.  With |X_k|_F <= min(a^k, 1.3 sqrt(m)) and |X_k|_2 <= 1.3, five steps leave at most
    2^-24 c 4.775 * 1.3 * sum_k a^(4 - k) min(a^k, 1.3 sqrt(m))
(705 x 705: 3.3e-5 of the result).  Products of 16 bits are off by 2^-18 of each term, rms 2^-19, of either sign: over K >= 705 terms 2^-19 /
sqrt(705) = 1.2 * 2^-24 of the norms of the rows, within c.  (X itself in 16 bits would leave 8e-5 to 6e-4 on the matrices below: that
rounding meets X directly.)  The rounding of a 16-bit result adds in quadrature, since the two have nothing to do with each other."""
import math

import pytest
import torch

import test_orthogonalize as T
from test_orthogonalize import check, gradient_like

# the entry point takes float32 coefficients and eps (include/dcc_ortho.h): 2^-25 of a coefficient is as much as the result's rounding
F32 = lambda x: float(torch.tensor(x, dtype=torch.float32))
COEFFS, EPS = tuple(F32(x) for x in (T.A, T.B, T.C)), F32(1e-7)


def reference(G, steps=5):
    return T.reference(G, steps, COEFFS, EPS)


def low_floor(M, N, dtype, seed=0):
    """a few strong directions over a low floor, which the steps raise to the same size"""
    gen = torch.Generator().manual_seed(seed)
    G = (torch.randn(M, 8, generator=gen) * torch.logspace(0, -2, 8)) @ torch.randn(8, N, generator=gen) + 1e-3 * torch.randn(M, N, generator=gen)
    return (1e-3 * G).to(dtype)


def rounded(ref, dtype):
    return float((ref.to(dtype).double() - ref).norm())


def by_steps(m, n, steps):
    a, k = 3.4445, (n + 127) // 128 * 128
    grown = sum(a ** (steps - 1 - i) * min(a ** i, 1.3 * math.sqrt(m)) for i in range(steps))
    return 2.0 ** -24 * (1 + math.sqrt(k / 96)) * 4.775 * 1.3 * grown


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 300), (2, 2), (31, 33), (65, 64), (96, 500), (500, 96), (256, 440), (384, 256), (256, 2704), (2704, 256),
                                   (40, 9001), (640, 700), (704, 705), (200, 16389), (16388, 200)], ids=lambda s: "%dx%d" % s)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("make", [gradient_like, low_floor])
def test_square_side(shape, dtype, make):
    import dcc_hip
    G = make(*shape, dtype=dtype, seed=shape[0])
    R = reference(G)
    off = float((dcc_hip.orthogonalize(G.cuda()).double().cpu() - R).norm())
    assert off <= rounded(R, dtype) * (1 + 4 / math.sqrt(R.numel())) + 1e-9 * float(R.norm()), "%.3e of %.3e" % (off, float(R.norm()))


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [1, 2, 5])
@pytest.mark.parametrize("shape", [(705, 705), (720, 901), (1030, 772)], ids=lambda s: "%dx%d" % s)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("make", [gradient_like, low_floor])
def test_step_by_step(shape, dtype, steps, make):
    import dcc_hip
    G = make(*shape, dtype=dtype, seed=shape[1])
    R = reference(G, steps)
    off = float((dcc_hip.orthogonalize(G.cuda(), steps=steps).double().cpu() - R).norm())
    room = math.hypot(rounded(R, dtype) * (1 + 4 / math.sqrt(R.numel())), by_steps(min(shape), max(shape), steps))
    assert off <= room, "%.3e, %.3e allowed (norm %.3e)" % (off, room, float(R.norm()))


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [10, 11, 16])
@pytest.mark.parametrize("shape", [(48, 64), (300, 48), (200, 16388), (720, 750)], ids=lambda s: "%dx%d" % s)
def test_many_steps(shape, steps):
    """three and four groups on the m x m side: X is formed in between, in two places in turn"""
    import dcc_hip
    G = gradient_like(*shape, seed=steps)
    check(dcc_hip.orthogonalize(G.cuda(), steps=steps), reference(G, steps), "%dx%d" % shape)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_mixed_list_of_more_than_one_launch(dtype):
    """small, long and step-by-step matrices in one list, more of each than a launch holds: the bits of single calls"""
    import dcc_hip
    kinds = [(705, 705), (50, 70), (200, 16389), (16389, 200), (128, 8201), (710, 720)]
    mats = [gradient_like(*kinds[i % 6], dtype=dtype, seed=i).cuda() for i in range(132)]
    got = dcc_hip.orthogonalize(mats)
    for i, (x, y) in enumerate(zip(mats, got)):
        assert torch.equal(dcc_hip.orthogonalize(x), y), (i, tuple(x.shape))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_step_by_step_in_a_graph(dtype):
    """captured once, replayed on other matrices with eager calls in between: what a call keeps in its workspace begins anew"""
    import dcc_hip
    shapes = [(720, 901), (901, 720), (60, 90)]
    sets = [[gradient_like(m, n, dtype=dtype, seed=10 * i + j).cuda() for j, (m, n) in enumerate(shapes)] for i in range(3)]
    buf = [x.clone() for x in sets[0]]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        dcc_hip.orthogonalize(buf)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = dcc_hip.orthogonalize(buf)
    for i in (1, 2, 1, 0):
        for x, y in zip(buf, sets[i]):
            x.copy_(y)
        graph.replay()
        got = [x.clone() for x in outs]
        torch.cuda.synchronize()
        for x, y in zip(got, dcc_hip.orthogonalize(sets[i])):
            assert torch.equal(x, y)
