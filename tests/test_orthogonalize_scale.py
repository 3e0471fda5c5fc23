"""The norm of an orthogonalised update at the ends of its range: zero with eps = 0, sums that leave float32 in either direction, on every path.

Bounds: those of tests/test_orthogonalize.py, since the scaled matrix is the same; a scaled input is an exact one (a power of two) wherever
no entry becomes subnormal, and where some do, the reference starts from the same subnormal entries."""
import pytest
import torch

from test_orthogonalize import check, gradient_like, reference

SHAPES = [(37, 50), (300, 200), (60, 33000), (720, 901), (901, 720)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "%dx%d" % s)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_zero_with_eps_zero(shape, dtype):
    """no gradient, no update: G == 0 gives 0 whatever eps is, and leaves the other matrices of the list alone"""
    import dcc_hip
    G = gradient_like(*shape, dtype=dtype).cuda()
    Z = torch.zeros_like(G)
    for eps in (0.0, 1e-45, 1e-7):
        z, x = dcc_hip.orthogonalize([Z, G], eps=eps)
        assert torch.equal(z, Z), eps
        check(x, reference(G, eps=float(torch.tensor(eps, dtype=torch.float32))))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "%dx%d" % s)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("power", [-120, -100, 100, 126])
def test_norms_outside_float32(shape, dtype, power):
    """|G|_F from 1e-38 to 1e41: its inverse is subnormal or infinite in float32"""
    import dcc_hip
    G = gradient_like(*shape, dtype=dtype, seed=5).double()
    G = (G / G.abs().max() * 2.0 ** power).to(dtype).cuda()
    assert torch.isfinite(G).all() and G.abs().max() > 0
    check(dcc_hip.orthogonalize(G, eps=0.0), reference(G, eps=0.0), "2^%d" % power)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "%dx%d" % s)
def test_subnormal_entries(shape):
    """every entry below 1e-38: a norm below float32's smallest normal number"""
    import dcc_hip
    G = gradient_like(*shape, seed=6).double()
    G = (G / G.norm() * 2.0 ** -128).float().cuda()        # some of the entries become 0
    check(dcc_hip.orthogonalize(G, eps=0.0), reference(G, eps=0.0))
