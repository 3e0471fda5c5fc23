"""The gated-delta recurrent core (algo_utils/rnn.GatedDeltaLayer, cfg.recurrent_core) and the Muon optimizer (algo_utils/optim.FlatMuon,
cfg.optimizer) as the policies use them: rollout step by step, update over sequences, whole training iterations."""
import math
import os
from argparse import Namespace

import numpy as np
import pytest
import torch
import yaml

from conftest import PKG

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _cfg(**over):
    cfg = {}
    for f in ("config/env_config/dcc.yaml", "config/algo_config/mappo.yaml", "config/expt.yaml"):
        cfg.update(yaml.safe_load(open(os.path.join(PKG, f))))
    cfg.update(over)
    return Namespace(**cfg)


def _layer(dev, N=2, H=24, heads=3, D=8):
    from algos.algo_utils.rnn import GatedDeltaLayer
    torch.manual_seed(3)
    lay = GatedDeltaLayer(H, H, N, True, heads, D)
    with torch.no_grad():
        for p in lay.parameters():
            p.add_(0.1 * torch.randn_like(p))
    return lay.to(dev)


def _data(dev, T=23, B=5, N=2, H=24, S=3 * 64):
    gen = torch.Generator().manual_seed(4)
    x = torch.randn(T * B, H, generator=gen)
    m = (torch.rand(T * B, 1, generator=gen) > 0.15).float()
    h = torch.randn(B, N, S, generator=gen)
    return [t.to(dev) for t in (x, h, m)]


@pytest.mark.parametrize("dev", DEVICES)
def test_sequence_equals_steps(dev):
    """the update's sequence call = the rollout's steps.  32-bit sums of at most 24 + 23 terms of order one, twice (two layers), after
    a LayerNorm: 100 roundings of 2^-24 on values of at most 4"""
    lay = _layer(dev)
    x, h, m = _data(dev)
    T, B = 23, 5
    seq, last = lay(x, h, m)
    outs, s = [], h
    with torch.no_grad():
        for t in range(T):
            o, s = lay(x[t * B:(t + 1) * B], s, m[t * B:(t + 1) * B])
            outs.append(o)
    assert float((torch.cat(outs) - seq).abs().max()) <= 100 * 2.0 ** -24 * 4
    assert float((s - last).abs().max()) <= 100 * 2.0 ** -24 * max(4.0, float(last.abs().max()))
    one, s1 = lay(x[:B], h, m[:B])                  # a step with gradients
    assert float((one - seq[:B]).abs().max()) <= 100 * 2.0 ** -24 * 4 and one.requires_grad and s1.shape == h.shape


@pytest.mark.parametrize("dev", DEVICES)
def test_gradients_of_the_layer(dev):
    """against the layer in float64 on the CPU; 200 roundings (a forward and a reversed recurrence) relative to each gradient's largest entry"""
    lay, ref = _layer(dev), _layer("cpu").double()
    x, h, m = _data(dev)
    xr, hr, mr = [t.double() for t in _data("cpu")]
    grads = []
    for l, a, s, k in ((lay, x, h, m), (ref, xr, hr, mr)):
        a, s = a.requires_grad_(True), s.requires_grad_(True)
        o, last = l(a, s, k)
        w = torch.linspace(-1, 1, o.numel(), dtype=torch.float64).view(o.shape).to(o)
        loss = (o * w).sum() + (last * last).sum() * 0.01
        grads.append([g.double().cpu() for g in torch.autograd.grad(loss, [a, s] + list(l.parameters()))])
    for g, r in zip(*grads):
        assert float((g - r).abs().max()) <= 200 * 2.0 ** -24 * max(1e-3, float(r.abs().max())) * 4


def test_restart_equals_a_fresh_sequence():
    lay = _layer("cpu")
    x, h, m = _data("cpu")
    B = 5
    m.fill_(1.0)
    m[10 * B:11 * B] = 0
    seq, last = lay(x, h, m)
    m2 = m[10 * B:].clone()
    part, last2 = lay(x[10 * B:], torch.zeros_like(h), m2)
    assert torch.allclose(seq[10 * B:], part, atol=1e-6) and torch.allclose(last, last2, atol=1e-6)


def test_configuration_keys():
    from algos.algo_utils.rnn import GatedDeltaLayer, RNNLayer, make_recurrent, state_size
    from algos.algo_utils.optim import FlatAdam, FlatMuon, make_optimizer
    cfg = _cfg()
    assert isinstance(make_recurrent(cfg), RNNLayer) and state_size(cfg) == cfg.algo_hidden_size
    cfg = _cfg(recurrent_core="gated_delta", delta_heads=2, delta_head_dim=8)
    assert isinstance(make_recurrent(cfg), GatedDeltaLayer) and state_size(cfg) == 128
    lin = torch.nn.Linear(16, 16)
    assert type(make_optimizer(_cfg(), lin.parameters(), lr=1e-3)) is FlatAdam
    assert type(make_optimizer(_cfg(optimizer="muon"), lin.parameters(), lr=1e-3)) is FlatMuon
    with pytest.raises(ValueError, match="recurrent_core"):
        make_recurrent(_cfg(recurrent_core="lstm"))
    with pytest.raises(ValueError, match="optimizer"):
        make_optimizer(_cfg(optimizer="sgd"), lin.parameters(), lr=1e-3)
    for kw in (dict(heads=0), dict(head_dim=0), dict(head_dim=129), dict(outputs_dim=8)):
        with pytest.raises(ValueError):
            GatedDeltaLayer(**dict(dict(inputs_dim=16, outputs_dim=16, recurrent_N=1, use_orthogonal=True), **kw))
    for kw in (dict(momentum=1.0), dict(ns_steps=0), dict(ns_steps=33)):
        with pytest.raises(ValueError):
            FlatMuon(lin.parameters(), **kw)


def _ns64(G, steps):
    X = G.T if G.shape[0] > G.shape[1] else G
    X = X / (X.norm() + 1e-7)
    for _ in range(steps):
        A = X @ X.T
        X = 3.4445 * X - 4.7750 * (A @ X) + 2.0315 * (A @ (A @ X))
    return X.T if G.shape[0] > G.shape[1] else X


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("max_norm,wd,nesterov", [(10.0, 0.0, True), (0.5, 0.01, True), (None, 0.02, False)])
def test_muon_step_against_float64(dev, max_norm, wd, nesterov):
    """three steps: matrices p <- (1 - lr wd) p - lr 0.2 sqrt(max(M, N)) NS(momentum), the rest Adam.  NS is held to 1e-4 of its norm
    (tests/test_orthogonalize.py derives 2^-24 * 141 * sqrt(m) = 1e-4 at m = 130), times the step; the rest to Adam's 1e-5 relative."""
    from algos.algo_utils.optim import FlatMuon
    torch.manual_seed(5)
    shapes = [(64, 37), (64,), (3, 50), (130, 64), (7,), (40, 300), (15, 200)]
    ps = [torch.nn.Parameter(torch.randn(*s).to(dev)) for s in shapes]
    opt = FlatMuon(ps, lr=1e-2, eps=1e-5, weight_decay=wd, nesterov=nesterov)
    P = [p.detach().double().cpu() for p in ps]
    M, V = [torch.zeros_like(p) for p in P], [torch.zeros_like(p) for p in P]
    for t in range(1, 4):
        opt.zero_grad()
        gs = [torch.randn(*s) for s in shapes]
        for p, g in zip(ps, gs):
            p.grad.add_(g.to(dev))
        n = opt.clip_and_step(max_norm)
        norm = math.sqrt(sum(float(g.double().square().sum()) for g in gs))
        assert abs(float(n) - norm) <= 1e-5 * norm
        clip = min(1.0, max_norm / (norm + 1e-6)) if max_norm else 1.0
        for i, g in enumerate(gs):
            g = g.double() * clip
            if P[i].dim() == 2 and min(P[i].shape) >= 16:
                M[i] = 0.95 * M[i] + g
                d = _ns64(g + 0.95 * M[i] if nesterov else M[i], 5)
                step = 1e-2 * 0.2 * math.sqrt(max(P[i].shape))
                P[i] = (1 - 1e-2 * wd) * P[i] - step * d
                room = step * 1e-4 * float(d.norm()) * t + 2.0 ** -24 * t * float(P[i].abs().max())
                assert float((ps[i].detach().double().cpu() - P[i]).abs().max()) <= room, shapes[i]
            else:
                g = g + wd * P[i]
                M[i] = 0.9 * M[i] + 0.1 * g
                V[i] = 0.999 * V[i] + 0.001 * g * g
                P[i] = P[i] - 1e-2 / (1 - 0.9 ** t) * M[i] / (V[i].sqrt() / math.sqrt(1 - 0.999 ** t) + 1e-5)
                assert torch.allclose(ps[i].detach().double().cpu(), P[i], rtol=1e-5, atol=1e-6), shapes[i]
    # checkpoint: a copy that takes over the state makes the same next step; Adam's checkpoint is refused
    from algos.algo_utils.optim import FlatAdam
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    other = FlatMuon(qs, lr=5.0, nesterov=nesterov)
    other.load_state_dict(opt.state_dict())
    for o, params in ((opt, ps), (other, qs)):
        o.zero_grad()
        for p, g in zip(params, gs):
            p.grad.add_(g.to(dev))
        o.clip_and_step(max_norm)
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))
    with pytest.raises(ValueError, match="another optimizer"):
        other.load_state_dict(FlatAdam([torch.nn.Parameter(p.detach().clone()) for p in ps]).state_dict())
    with pytest.raises(ValueError, match="another optimizer"):
        FlatAdam([torch.nn.Parameter(p.detach().clone()) for p in ps]).load_state_dict(opt.state_dict())


def test_muon_without_matrices_is_adam_and_without_vectors_runs():
    from algos.algo_utils.optim import FlatAdam, FlatMuon
    torch.manual_seed(1)
    v = torch.randn(9)
    a, b = [torch.nn.Parameter(v.clone())], [torch.nn.Parameter(v.clone())]
    oa, ob = FlatAdam(a, lr=1e-2), FlatMuon(b, lr=1e-2)
    for o, p in ((oa, a), (ob, b)):
        p[0].grad.add_(torch.arange(9.0))
        o.clip_and_step(1.0)
    assert torch.equal(a[0], b[0])
    w = [torch.nn.Parameter(torch.randn(20, 20))]
    o = FlatMuon(w, lr=1e-2)
    before = w[0].detach().clone()
    w[0].grad.add_(torch.randn(20, 20))
    o.step()
    assert not torch.equal(before, w[0])


@pytest.mark.gpu
def test_momentum_and_apply_refuse():
    import dcc_hip
    x = torch.zeros(64, device="cuda")
    for bad in (lambda: dcc_hip.muon_momentum(x, x[:32], x.clone(), 0.9), lambda: dcc_hip.muon_momentum(x, x.clone(), x.clone().double(), 0.9),
                lambda: dcc_hip.muon_momentum(x[1:], x[1:].clone(), x[1:].clone(), 0.9), lambda: dcc_hip.muon_apply(x, x[:32], []),
                lambda: dcc_hip.muon_apply(x, x.clone(), [(0, 65, 1.0)]), lambda: dcc_hip.muon_apply(x, x.clone(), [(0, 8, 1.0), (4, 8, 1.0)]),
                lambda: dcc_hip.muon_apply(x, x.clone(), [(2, 8, 1.0)]), lambda: dcc_hip.muon_apply(x, x.clone(), [(-4, 8, 1.0)])):
        with pytest.raises((ValueError, dcc_hip.DccError)):
            bad()
    dcc_hip.muon_apply(x, torch.ones_like(x), [(0, 5, 1.0), (8, 0, 1.0), (12, 3, 2.0)], 0.5)
    want = torch.zeros(64); want[:5] = -1; want[12:15] = -2
    assert torch.equal(x.cpu(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["use_recurrent_policy", "use_naive_recurrent_policy"])
def test_training_with_the_delta_core_and_muon(mode, tmp_path):
    """rollouts step by step, updates over chunks / whole episodes with 2 mini-batches, evaluation, checkpoint and resume"""
    import utils.pytorch_utils as ptu
    ptu.set_gpu_mode(True, 0)
    from learner import Learner
    kw = dict(n_rollout_threads=12, n_eval_rollout_threads=0, num_agents=4, num_pois=16, max_ep_len=40, n_iters=4, ppo_epoch=2,
              algo_hidden_size=32, save_model=False, num_mini_batch=2, data_chunk_length=5, use_hip_graph=False, recurrent_core="gated_delta",
              delta_heads=2, delta_head_dim=16, optimizer="muon", recurrent_N=2, **{mode: True})
    lr = Learner(_cfg(**kw))
    b = lr.rl_buffer
    assert b.rnn_states.shape == (41, 12, 4, 2, 512)
    before = [p.detach().clone() for p in lr.policy.actor.parameters()]
    for _ in range(2):
        r = lr.rollout(b, lr.train_envs)
        info = lr.rl_update()
        assert np.isfinite(r["reward"]) and all(np.isfinite(v) for v in info.values())
    assert float(b.rnn_states[1:].abs().sum()) > 0
    done_next = b.masks[1:, :, :, 0] == 0
    assert float(b.rnn_states[1:][done_next].abs().sum()) == 0.0
    moved = [not torch.equal(p, q) for p, q in zip(before, lr.policy.actor.parameters())]
    assert all(moved)
    # the update's forward pass sees what the rollout saw: the first PPO ratio of a fresh batch is 1.  exp of a difference of two
    # log-probs of size <= 10 computed by two orders of the same sums (40 steps, 2 layers): 1e-4
    lr.rollout(b, lr.train_envs)
    adv = lr.trainer.normalized_advantages(b)
    gen = b.recurrent_generator(adv, 1, 5) if mode == "use_recurrent_policy" else b.naive_recurrent_generator(adv, 1)
    with torch.no_grad():
        ratio = lr.trainer._forward_losses(next(gen))[3]
    assert abs(float(ratio.mean()) - 1.0) <= 1e-4
    lr.rl_update()
    path = str(tmp_path / "ck.pt")
    lr.save_checkpoint(path)
    lr2 = Learner(_cfg(**kw))
    lr2.load_checkpoint(path)
    for l in (lr, lr2):
        l.warmup(l.rl_buffer, l.train_envs)
        torch.manual_seed(5)
        l.rollout(l.rl_buffer, l.train_envs)
        l.rl_update()
    for p, q in zip(lr.policy.actor.parameters(), lr2.policy.actor.parameters()):
        assert torch.equal(p, q)
    res = lr.evaluate(steps=10)
    assert 0.0 <= res["coverage_rate"] <= 1.0
    ptu.set_gpu_mode(False)


@pytest.mark.gpu
def test_muon_trains_the_shipped_policy():
    """optimizer: muon with the feed-forward, state-only default (hipGraph rollouts read parameters that the step moves in place)"""
    import utils.pytorch_utils as ptu
    ptu.set_gpu_mode(True, 0)
    from learner import Learner
    lr = Learner(_cfg(n_rollout_threads=16, n_eval_rollout_threads=0, max_ep_len=30, n_iters=3, ppo_epoch=2, save_model=False, optimizer="muon"))
    for _ in range(3):
        r = lr.rollout(lr.rl_buffer, lr.train_envs)
        info = lr.rl_update()
        assert np.isfinite(r["reward"]) and all(np.isfinite(v) for v in info.values())
    mats = [p for p, _ in lr.policy.actor_optimizer._mats]
    assert [tuple(p.shape) for p in mats] == [(256, 110), (256, 256)]
    ptu.set_gpu_mode(False)
