"""States of the recurrent policies on their way through learner and buffer: restarts are selected, and a buffer that cannot fit says so."""
from types import SimpleNamespace

import pytest
import torch

NAN, INF = float("nan"), float("inf")


def test_a_finished_env_restarts_whatever_its_state_held():
    from learner import Learner
    E, N, L, S = 3, 2, 1, 5
    rnn_a, rnn_c = torch.randn(E, N, L, S), torch.randn(E, N, L, S)
    rnn_a[1, 0, 0, 2], rnn_c[1, 1, 0, 0], rnn_c[1, 0, 0, 1] = NAN, INF, -INF
    kept = []
    buf = SimpleNamespace(n_rollout_threads=E, insert=lambda *a: kept.append(a))
    done = torch.tensor([0, 1, 0], dtype=torch.uint8)
    Learner.insert(SimpleNamespace(n_agents=N), ({"done": done, "reward": torch.zeros(E)}, None, None, None, rnn_a, rnn_c), buf)
    a, c, masks = kept[0][2], kept[0][3], kept[0][-1]
    assert (a[1] == 0).all() and (c[1] == 0).all()
    for e in (0, 2):
        assert torch.equal(a[e], rnn_a[e]) and torch.equal(c[e], rnn_c[e])
    assert masks.shape == (E, N, 1) and float(masks[1].sum()) == 0 and float(masks.sum()) == (E - 1) * N


def test_states_that_cannot_fit_are_refused_by_name():
    """the buffer keeps every step's state, twice; 4096 envs of 8 agents with 4 heads of 64 x 64 need 648 GB and one card has 288"""
    from buffer.shared_buffer import check_state_memory, recurrent_state_bytes
    one = 151 * 4096 * 8 * 1 * 4 * 64 * 64 * 4
    assert recurrent_state_bytes(150, 4096, 8, 1, 4 * 64 * 64) == 2 * one
    with pytest.raises(ValueError, match="648.5 GB.*delta_head_dim"):
        check_state_memory(2 * one, 288 * 10 ** 9)
    check_state_memory(recurrent_state_bytes(150, 4096, 8, 1, 4 * 32 * 32), 288 * 10 ** 9)       # 162 GB: the default heads
    check_state_memory(recurrent_state_bytes(150, 4096, 8, 1, 256), 288 * 10 ** 9)


@pytest.mark.gpu
def test_layer_in_float64_steps_on_the_device():
    """a step without gradients of a layer that the kernels don't take runs in torch, like its sequence"""
    from algos.algo_utils.rnn import GatedDeltaLayer
    torch.manual_seed(1)
    lay = GatedDeltaLayer(24, 24, 2, True, 3, 8).double()
    x, h, m = torch.randn(5, 24).double(), torch.randn(5, 2, 3 * 64).double(), torch.tensor([1, 0, 1, 1, 1]).double().view(5, 1)
    with torch.no_grad():
        want = lay(x, h, m)
        got = lay.cuda()(x.cuda(), h.cuda(), m.cuda())
    for a, b in zip(want, got):
        assert torch.allclose(a, b.cpu(), rtol=1e-6, atol=1e-6)            # masks pass through float32; they are 0 and 1


@pytest.mark.gpu
def test_sequence_takes_masks_of_any_type_and_other_gates_in_torch():
    from algos.algo_utils import fused
    from test_gated_delta import NAMES, bound, make
    d = make(20, 3, 1, 2, 16, 24, reset=0.3, seed=4, device="cuda")
    o, S = fused.gated_delta(*[d[n] for n in NAMES], d["masks"])
    for masks in (d["masks"].bool(), d["masks"].to(torch.int32), d["masks"].double()):
        o2, S2 = fused.gated_delta(*[d[n] for n in NAMES], masks)
        assert torch.equal(o, o2) and torch.equal(S, S2)
    args = [d[n].double() if n in ("g", "beta", "state") else d[n] for n in NAMES]
    o2, S2 = fused.gated_delta(*args, d["masks"])
    assert o2.dtype == torch.float32
    assert float((o2 - o).abs().max()) <= 2 * bound(20, 16) * float(o.abs().max()) and float((S2 - S).abs().max()) <= 2 * bound(20, 16) * float(S.abs().max())
