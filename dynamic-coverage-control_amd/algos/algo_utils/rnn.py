"""GRU + LayerNorm layer of the recurrent policy variants (reference: uav_dcc_control/algos/algo_utils/rnn.py:7-82;
used by R_Actor / R_Critic when `use_recurrent_policy` or `use_naive_recurrent_policy` is set -- both are off in
the shipped mappo.yaml).  Same parameters and names (`rnn.weight_ih_l0`, ..., `norm.weight`) and the same function:

  * one step (rollout):   x [B,H], hxs [B,recurrent_N,H], masks [B,1]  ->  GRU(x, hxs * mask)
  * a sequence (update):  x [T*B,H] (time-major flattening), hxs [B,recurrent_N,H] = state at t=0, masks [T*B,1]

The reference cuts the sequence at the steps where any mask is 0 and runs one multi-step GRU call per segment; to find
the cut points it copies the masks to the host (`.nonzero().cpu()`: a device synchronisation inside every PPO
mini-batch).  Multiplying the state by the step's mask before EVERY step is the same arithmetic (the mask is exactly
1.0 inside a segment) and needs no host round trip, so the update stays asynchronous on the device.

`GatedDeltaLayer` (cfg.recurrent_core: gated_delta) stands in for the GRU with the same call: its state is a matrix per head instead of a
vector, and a sequence is one launch forward and one backward (include/dcc_delta.h) where the GRU steps through it in Python.
"""
import torch
import torch.nn as nn
import torch.nn.functional as F

from . import fused


class RNNLayer(nn.Module):
    def __init__(self, inputs_dim, outputs_dim, recurrent_N, use_orthogonal):
        super().__init__()
        self._recurrent_N = recurrent_N
        self.rnn = nn.GRU(inputs_dim, outputs_dim, num_layers=recurrent_N)
        for name, param in self.rnn.named_parameters():   # rnn.py:15-22
            if "bias" in name:
                nn.init.constant_(param, 0)
            elif "weight" in name:
                (nn.init.orthogonal_ if use_orthogonal else nn.init.xavier_uniform_)(param)
        self.norm = nn.LayerNorm(outputs_dim)

    def forward(self, x, hxs, masks):
        B = hxs.size(0)
        h = hxs.transpose(0, 1).contiguous()                       # [recurrent_N, B, H]
        if x.size(0) == B:
            out, h = self.rnn(x.unsqueeze(0), h * masks.view(1, B, 1))
            x = out.squeeze(0)
        else:
            T = x.size(0) // B
            xs, ms = x.view(T, B, -1), masks.view(T, 1, B, 1)
            outs = []
            for t in range(T):
                out, h = self.rnn(xs[t:t + 1], h * ms[t])
                outs.append(out)
            x = torch.cat(outs, dim=0).reshape(T * B, -1)
        return self.norm(x), h.transpose(0, 1)


class GatedDeltaLayer(nn.Module):
    """`recurrent_N` residual gated-delta layers + LayerNorm, called like RNNLayer with states of heads * head_dim^2 numbers:
        q, k, v, a, b = W x;   q, k of unit length;   g = -exp(A_log) softplus(a + dt_bias);   beta = sigmoid(b)
        x <- x + W_o RMSNorm(gated_delta(q, k, v, g, beta))
    masks restart the state (0: the episode ended before this step)."""

    def __init__(self, inputs_dim, outputs_dim, recurrent_N, use_orthogonal, heads=4, head_dim=32):
        super().__init__()
        if inputs_dim != outputs_dim:
            raise ValueError("GatedDeltaLayer: the residual path needs inputs_dim == outputs_dim")
        if not (1 <= heads and 1 <= head_dim <= 128):
            raise ValueError("GatedDeltaLayer: heads >= 1 and 1 <= head_dim <= 128")
        self._recurrent_N, self.heads, self.head_dim = recurrent_N, heads, head_dim
        w = heads * head_dim
        init = nn.init.orthogonal_ if use_orthogonal else nn.init.xavier_uniform_
        self.qkv, self.gates, self.out = nn.ModuleList(), nn.ModuleList(), nn.ModuleList()
        self.A_log, self.dt_bias, self.scale = nn.ParameterList(), nn.ParameterList(), nn.ParameterList()
        for _ in range(recurrent_N):
            self.qkv.append(nn.Linear(inputs_dim, 3 * w, bias=False))
            self.gates.append(nn.Linear(inputs_dim, 2 * heads))
            self.out.append(nn.Linear(w, outputs_dim, bias=False))
            for lin in (self.qkv[-1], self.gates[-1], self.out[-1]):
                init(lin.weight)
            nn.init.constant_(self.gates[-1].bias, 0)
            # time constants of the heads: decay 1/2 .. 1/64 per step where the gate is at its bias
            dt = torch.logspace(-1, -6, heads, base=2.0) if heads > 1 else torch.tensor([0.1])
            self.A_log.append(nn.Parameter(torch.zeros(heads)))
            self.dt_bias.append(nn.Parameter(torch.log(torch.expm1(dt))))
            self.scale.append(nn.Parameter(torch.ones(head_dim)))
        self.norm = nn.LayerNorm(outputs_dim)

    def forward(self, x, hxs, masks):
        B, H, D = hxs.size(0), self.heads, self.head_dim
        T = x.size(0) // B
        m = masks.reshape(T, B).float()
        states = []
        for i in range(self._recurrent_N):
            q, k, v = self.qkv[i](x).view(T, B, 3, H, D).unbind(2)
            a, b = self.gates[i](x).view(T, B, 2, H).unbind(2)
            q, k = F.normalize(q, dim=-1), F.normalize(k, dim=-1)
            g = -torch.exp(self.A_log[i]) * F.softplus(a + self.dt_bias[i])
            beta = torch.sigmoid(b)
            S = hxs[:, i].reshape(B, H, D, D)
            if T == 1 and x.is_cuda and x.dtype == torch.float32 and not torch.is_grad_enabled() and not torch.is_autocast_enabled():
                import dcc_hip
                o, S = dcc_hip.gated_delta_step(q[0], k[0], v[0], g[0], beta[0], S.contiguous(), m[0])
            else:
                o, S = fused.gated_delta(q, k, v, g, beta, S, m)
            o = o.view(T * B, H, D)
            o = o * torch.rsqrt(o.square().mean(-1, keepdim=True) + 1e-6) * self.scale[i]
            x = x + self.out[i](o.view(T * B, H * D))
            states.append(S.reshape(B, H * D * D))
        return self.norm(x), torch.stack(states, 1)


CORES = ("gru", "gated_delta")


def _core(cfg):
    name = getattr(cfg, "recurrent_core", "gru")
    if name not in CORES:
        raise ValueError("recurrent_core: %r is not one of %s" % (name, list(CORES)))
    return name


def make_recurrent(cfg):
    """The recurrent core that cfg names, between trunk and head."""
    H = cfg.algo_hidden_size
    if _core(cfg) == "gru":
        return RNNLayer(H, H, cfg.recurrent_N, cfg.use_orthogonal)
    return GatedDeltaLayer(H, H, cfg.recurrent_N, cfg.use_orthogonal, int(getattr(cfg, "delta_heads", 4)), int(getattr(cfg, "delta_head_dim", 32)))


def state_size(cfg):
    """Numbers of recurrent state per row and layer (the last axis of hxs)."""
    if _core(cfg) == "gru":
        return cfg.algo_hidden_size
    return int(getattr(cfg, "delta_heads", 4)) * int(getattr(cfg, "delta_head_dim", 32)) ** 2
