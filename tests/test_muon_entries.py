"""Refusals of the element-wise ends of a Muon step (include/dcc_ortho.h): clips that are no device number, arrays over each other."""
import pytest
import torch


def test_muon_momentum_checks_its_clip_and_its_arrays():
    """a clip that is no number on the device would be read through a host address"""
    import dcc_hip
    for bad in (0.5, torch.tensor(0.5), torch.tensor([0.5], dtype=torch.float64), torch.empty(0)):
        with pytest.raises(ValueError, match="clip"):
            dcc_hip.check_clip("muon_momentum", bad, torch.device("cuda", 0))
    dcc_hip.check_clip("muon_momentum", None, torch.device("cuda", 0))


def test_muon_entries_refuse_arrays_over_each_other():
    import ctypes
    import dcc_hip
    L = dcc_hip.load_library()
    buf = (ctypes.c_float * 4096)()
    a = (ctypes.addressof(buf) + 63) // 64 * 64
    go = lambda g, b, d, n=64: L.dcc_muon_momentum(g, b, d, n, 0.9, 1, None, None)
    for g, b, d in ((a, a, a + 1024), (a, a + 1024, a), (a, a + 1024, a + 1024), (a, a + 1024, a + 1024 + 240), (a + 240, a + 1024, a)):
        assert go(g, b, d) == -1 and b"apart" in L.dcc_last_error()
    seg = (dcc_hip.MuonSeg * 1)(dcc_hip.MuonSeg(0, 64, 1.0))
    for d in (a, a + 16, a + 240):
        assert L.dcc_muon_apply(a, d, seg, 1, 1.0, None) == -1 and b"apart" in L.dcc_last_error()


@pytest.mark.gpu
def test_muon_momentum_refuses_on_the_device():
    import dcc_hip
    x, y, z = (torch.zeros(64, device="cuda") for _ in range(3))
    for clip in (0.5, torch.tensor(0.5), torch.tensor(0.5, device="cuda", dtype=torch.float64)):
        with pytest.raises(ValueError, match="clip"):
            dcc_hip.muon_momentum(x, y, z, 0.9, True, clip)
        with pytest.raises(ValueError, match="clip"):
            dcc_hip.adam_step(x, y, z, z.clone(), 1e-3, 1.0, 0.9, 0.99, 1e-8, 0.0, clip)
    with pytest.raises(dcc_hip.DccError, match="apart"):
        dcc_hip.muon_momentum(x, y, y, 0.9)
    with pytest.raises(dcc_hip.DccError, match="apart"):
        dcc_hip.muon_apply(x, x, [(0, 8, 1.0)])
    dcc_hip.muon_momentum(x + 1, y, z, 0.5, True, torch.full((), 0.5, device="cuda"))
    assert (y == 0.5).all() and (z == 0.75).all()
