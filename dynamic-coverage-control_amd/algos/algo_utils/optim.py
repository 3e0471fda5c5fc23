"""Adam + gradient-norm clipping on FLAT parameter storage (include/dcc_optim.h).

The reference builds two `torch.optim.Adam` (uav_dcc_control/algos/mappo.py:27-37) and, per PPO step and network, calls
`nn.utils.clip_grad_norm_` then `.step()` (mappo.py:176-185).  Same update rule here, different storage:

  * all parameters of a network are views into ONE flat float32 array (each starting on a 256-byte boundary), their
    `.grad` are views into a second one, the Adam moments are two more;
  * `clip_and_step(max_norm)` is three HIP launches (norm partials, clip coefficient, Adam) instead of ~25 small torch
    launches, with no host synchronisation -- the clip coefficient never leaves the device;
  * `zero_grad()` is one memset, and the multi-GPU path all-reduces `flat_grad` directly (no cat / copy-back).

`FlatMuon` (cfg.optimizer: muon) keeps the same storage and entry points and trains the weight matrices with orthogonalised updates.

On a CPU device (the gloo / golden tests of the host logic) the same arithmetic runs as a handful of torch ops on the
flat arrays; on a HIP device the kernels are mandatory (dcc_hip raises if libdcc_hip.so is missing).
"""
import math

import torch

_ALIGN = 64     # floats: every parameter view starts 256-byte aligned (float4 kernels, GEMM operands)


class FlatAdam(torch.optim.Optimizer):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0):
        params = list(params)
        if not params:
            raise ValueError("FlatAdam: no parameters")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        dev, dt = params[0].device, params[0].dtype
        if dt != torch.float32 or any(p.device != dev or p.dtype != dt for p in params):
            raise ValueError("FlatAdam: float32 parameters on one device")
        self._params = params
        self._numels = [p.numel() for p in params]
        self._offsets, n = [], 0
        for p in params:
            self._offsets.append(n)
            n += (p.numel() + _ALIGN - 1) // _ALIGN * _ALIGN
        self.numel = n
        self.flat_param = torch.zeros(n, dtype=dt, device=dev)
        self.flat_grad = torch.zeros(n, dtype=dt, device=dev)
        self.exp_avg = torch.zeros(n, dtype=dt, device=dev)
        self.exp_avg_sq = torch.zeros(n, dtype=dt, device=dev)
        with torch.no_grad():
            for p, off in zip(params, self._offsets):
                view = self.flat_param[off:off + p.numel()].view_as(p)
                view.copy_(p)
                p.data = view                                            # the module's parameter now IS the view
                p.grad = self.flat_grad[off:off + p.numel()].view_as(p)   # autograd accumulates in place into the view
        self.step_count = 0
        self._norm_out = torch.zeros(2, dtype=dt, device=dev)           # {grad norm, clip coefficient}
        self._ws = None

    # padding between the views stays zero: zero gradient, zero moments -> Adam leaves it at zero

    def _check_views(self):
        """Every parameter must still BE its view into flat_param: the kernels update flat_param through raw pointers, so a
        parameter whose storage was moved behind the optimizer's back (module.to(...) / any nn.Module._apply -- which also
        makes nn.GRU.flatten_parameters() re-allocate its weights --, load_state_dict(assign=True), p.data = ...) would keep
        computing with a detached tensor while the optimizer trains the orphaned view: training stalls silently.  Host-side
        pointer compare only (no sync).  A moved parameter of unchanged shape / dtype / device is re-attached -- its
        current values, the ones the network computes with, are copied into the view; anything else raises.  Do not call
        .to() on a network after its optimizer was built."""
        base = self.flat_param.data_ptr()
        for p, off, numel in zip(self._params, self._offsets, self._numels):
            if p.data_ptr() == base + 4 * off:
                continue
            view = self.flat_param[off:off + numel]
            if p.device != view.device or p.dtype != view.dtype or p.numel() != numel:
                raise RuntimeError("FlatAdam: a parameter left the optimizer's flat storage and changed device / dtype / size "
                                   "(%s %s, expected %s %s); rebuild the optimizer after moving a network"
                                   % (p.device, p.dtype, view.device, view.dtype))
            with torch.no_grad():
                view.copy_(p.data.reshape(-1))
                p.data = view.view(p.shape)

    def zero_grad(self, set_to_none=False):
        """One memset; the .grad views are re-attached if a caller dropped them (set_to_none elsewhere), and so are
        parameters that left the flat storage (_check_views)."""
        self._check_views()
        self.flat_grad.zero_()
        for p, off in zip(self._params, self._offsets):
            g = p.grad
            if g is None or g.data_ptr() != self.flat_grad.data_ptr() + 4 * off:
                p.grad = self.flat_grad[off:off + p.numel()].view_as(p)

    def _lr(self):
        return float(self.param_groups[0]["lr"])

    @torch.no_grad()
    def clip_and_step(self, max_norm=None):
        """clip_grad_norm_(params, max_norm) (None / <= 0: norm only) followed by one Adam step.  Returns the gradient
        norm BEFORE clipping as a 0-d device tensor (no sync)."""
        self._check_views()
        g = self.param_groups[0]
        beta1, beta2 = g["betas"]
        self.step_count += 1
        t = self.step_count
        step_size = self._lr() / (1.0 - beta1 ** t)
        bc2_sqrt = math.sqrt(1.0 - beta2 ** t)
        mn = float(max_norm) if max_norm else 0.0
        if self.flat_param.is_cuda:
            import dcc_hip
            if self._ws is None:
                self._ws = torch.empty(dcc_hip.grad_norm_workspace_floats(self.numel), dtype=torch.float32, device=self.flat_param.device)
            dcc_hip.grad_norm_clip(self.flat_grad, mn, self._norm_out, self._ws)
            dcc_hip.adam_step(self.flat_param, self.flat_grad, self.exp_avg, self.exp_avg_sq, step_size, bc2_sqrt, beta1, beta2,
                              g["eps"], g["weight_decay"], self._norm_out[1:])
            return self._norm_out[0].clone()
        norm = torch.linalg.vector_norm(self.flat_grad)
        clip = torch.clamp(mn / (norm + 1e-6), max=1.0) if mn > 0 else torch.ones((), dtype=norm.dtype)
        gr = self.flat_grad * clip
        if g["weight_decay"] != 0:
            gr = gr + g["weight_decay"] * self.flat_param
        self.exp_avg.lerp_(gr, 1.0 - beta1)
        self.exp_avg_sq.mul_(beta2).addcmul_(gr, gr, value=1.0 - beta2)
        denom = (self.exp_avg_sq.sqrt() / bc2_sqrt).add_(g["eps"])
        self.flat_param.addcdiv_(self.exp_avg, denom, value=-step_size)
        return norm

    def step(self, closure=None):
        self.clip_and_step(None)

    # ---- checkpoints -----------------------------------------------------------------------------------------------------
    FORMAT = "flat_adam_v1"

    def state_dict(self):
        return {"format": self.FORMAT, "step": self.step_count, "exp_avg": self.exp_avg.detach().cpu().clone(),
                "exp_avg_sq": self.exp_avg_sq.detach().cpu().clone(), "offsets": list(self._offsets),
                "numels": [p.numel() for p in self._params],
                "param_groups": [{k: v for k, v in g.items() if k != "params"} for g in self.param_groups]}

    def load_state_dict(self, sd):
        """This optimizer's own state, or (FlatAdam) that of a torch.optim.Adam.  Anything else is refused with nothing changed."""
        if sd.get("format") == self.FORMAT:
            if sd["numels"] != [p.numel() for p in self._params]:
                raise ValueError("%s.load_state_dict: parameter layout differs" % type(self).__name__)
            self.exp_avg.copy_(sd["exp_avg"]); self.exp_avg_sq.copy_(sd["exp_avg_sq"])
            self.step_count = int(sd["step"])
            for g, sg in zip(self.param_groups, sd["param_groups"]):
                g.update({k: v for k, v in sg.items() if k != "params"})
            return
        # (without a format: a torch.optim.Adam's, in the order that FlatAdam keeps; FlatMuon reorders, and its exp_avg is no average)
        if "format" in sd or self.FORMAT != FlatAdam.FORMAT:
            raise ValueError("%s.load_state_dict: the checkpoint holds the state of another optimizer (%s)"
                             % (type(self).__name__, sd.get("format", "torch.optim.Adam")))
        # a torch.optim.Adam state_dict (checkpoints written before the flat optimizer): per-parameter moments
        state, groups = sd["state"], sd["param_groups"]
        ids = [i for g in groups for i in g["params"]]
        if len(ids) != len(self._params):
            raise ValueError("FlatAdam.load_state_dict: %d parameters in the checkpoint, %d here" % (len(ids), len(self._params)))
        for i, p in zip(ids, self._params):
            for m in ("exp_avg", "exp_avg_sq") if state.get(i) is not None else ():
                if state[i][m].shape != p.shape:
                    raise ValueError("FlatAdam.load_state_dict: parameter %s is %s here, its %s in the checkpoint %s"
                                     % (i, tuple(p.shape), m, tuple(state[i][m].shape)))
        self.exp_avg.zero_(); self.exp_avg_sq.zero_()
        step = 0
        for i, p, off in zip(ids, self._params, self._offsets):
            st = state.get(i)
            if st is None:
                continue
            self.exp_avg[off:off + p.numel()].copy_(st["exp_avg"].reshape(-1))
            self.exp_avg_sq[off:off + p.numel()].copy_(st["exp_avg_sq"].reshape(-1))
            step = max(step, int(float(st["step"])))
        self.step_count = step
        for g, sg in zip(self.param_groups, groups):
            g.update({k: sg[k] for k in ("lr", "betas", "eps", "weight_decay") if k in sg})


NEWTON_SCHULZ = (3.4445, -4.7750, 2.0315)


class FlatMuon(FlatAdam):
    """Muon on the same flat storage (include/dcc_ortho.h): the update of every weight matrix is its Nesterov momentum with all
    singular values drawn towards 1 by Newton-Schulz products; vectors and narrow heads keep Adam.

      * matrix parameters (2-D, both sides >= MIN_SIDE) lie behind all others in the flat arrays: one Adam launch on the front, one
        momentum launch, one `orthogonalize` of the whole list and one launch that applies it on the back;
      * the step of an [M, N] matrix is lr * RMS * sqrt(max(M, N)) times the orthogonalised momentum: its entries then have the root mean
        square RMS * lr, about Adam's, so that both halves share lr and its schedule;
      * clip_grad_norm_ is taken over all gradients before either half, like FlatAdam's; weight_decay is decoupled for the matrices
        (p *= 1 - lr * weight_decay), Adam's own for the rest; the momentum lives in exp_avg."""
    MIN_SIDE = 16
    RMS = 0.2
    FORMAT = "flat_muon_v1"

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, momentum=0.95, nesterov=True, ns_steps=5):
        params = list(params)
        if not 0.0 <= momentum < 1.0:
            raise ValueError("FlatMuon: momentum must lie in [0, 1)")
        if not 1 <= int(ns_steps) <= 32:
            raise ValueError("FlatMuon: ns_steps must lie in 1..32")
        matrix = [p.dim() == 2 and min(p.shape) >= self.MIN_SIDE for p in params]
        super().__init__([p for p, m in zip(params, matrix) if not m] + [p for p, m in zip(params, matrix) if m],
                         lr=lr, betas=betas, eps=eps, weight_decay=weight_decay)
        for g in self.param_groups:
            g.update(momentum=float(momentum), nesterov=bool(nesterov), ns_steps=int(ns_steps))
        self._n_adam = self._offsets[len(params) - sum(matrix)] if any(matrix) else self.numel
        self._mats = [(p, off - self._n_adam) for p, off, in zip(self._params, self._offsets) if off >= self._n_adam]
        n = self.numel - self._n_adam
        self._dir = torch.zeros(n, dtype=torch.float32, device=self.flat_param.device)
        self._ortho = torch.zeros(n, dtype=torch.float32, device=self.flat_param.device)
        views = lambda flat: [flat[o:o + p.numel()].view(p.shape) for p, o in self._mats]
        self._dir_views, self._ortho_views = views(self._dir), views(self._ortho)

    @torch.no_grad()
    def clip_and_step(self, max_norm=None):
        """clip_grad_norm_(params, max_norm) (None / <= 0: norm only), then one Muon step on the matrices and one Adam step on the rest.
        Returns the gradient norm BEFORE clipping as a 0-d device tensor (no sync)."""
        self._check_views()
        g = self.param_groups[0]
        beta1, beta2 = g["betas"]
        self.step_count += 1
        t, lr, cut = self.step_count, self._lr(), self._n_adam
        step_size, bc2_sqrt = lr / (1.0 - beta1 ** t), math.sqrt(1.0 - beta2 ** t)
        mn = float(max_norm) if max_norm else 0.0
        segs = [(o, p.numel(), lr * self.RMS * math.sqrt(max(p.shape))) for p, o in self._mats]
        keep = 1.0 - lr * g["weight_decay"]
        front = [a[:cut] for a in (self.flat_param, self.flat_grad, self.exp_avg, self.exp_avg_sq)]
        p_back, g_back, m_back = (a[cut:] for a in (self.flat_param, self.flat_grad, self.exp_avg))
        if self.flat_param.is_cuda:
            import dcc_hip
            if self._ws is None:
                self._ws = torch.empty(dcc_hip.grad_norm_workspace_floats(self.numel), dtype=torch.float32, device=self.flat_param.device)
            dcc_hip.grad_norm_clip(self.flat_grad, mn, self._norm_out, self._ws)
            if cut:
                dcc_hip.adam_step(*front, step_size, bc2_sqrt, beta1, beta2, g["eps"], g["weight_decay"], self._norm_out[1:])
            if self._mats:
                dcc_hip.muon_momentum(g_back, m_back, self._dir, g["momentum"], g["nesterov"], self._norm_out[1:])
                dcc_hip.orthogonalize(self._dir_views, steps=g["ns_steps"], coeffs=NEWTON_SCHULZ, out=self._ortho_views)
                dcc_hip.muon_apply(p_back, self._ortho, segs, keep)
            return self._norm_out[0].clone()
        norm = torch.linalg.vector_norm(self.flat_grad)
        clip = torch.clamp(mn / (norm + 1e-6), max=1.0) if mn > 0 else torch.ones((), dtype=norm.dtype)
        if cut:
            p, gr, m, v = front
            gr = gr * clip
            if g["weight_decay"] != 0:
                gr = gr + g["weight_decay"] * p
            m.lerp_(gr, 1.0 - beta1)
            v.mul_(beta2).addcmul_(gr, gr, value=1.0 - beta2)
            p.addcdiv_(m, (v.sqrt() / bc2_sqrt).add_(g["eps"]), value=-step_size)
        if self._mats:
            gr = g_back * clip
            m_back.mul_(g["momentum"]).add_(gr)
            self._dir.copy_(gr + g["momentum"] * m_back if g["nesterov"] else m_back)
            for (o, n, scale), d in zip(segs, self._dir_views):
                p_back[o:o + n].mul_(keep).sub_(scale * _newton_schulz(d, g["ns_steps"]).reshape(-1))
        return norm


def _newton_schulz(G, steps, coeffs=NEWTON_SCHULZ, eps=1e-7):
    """The orthogonalised update in plain torch (host logic on the CPU)."""
    a, b, c = coeffs
    X = G.t() if G.shape[0] > G.shape[1] else G
    X = X / (X.norm() + eps)
    for _ in range(steps):
        A = X @ X.t()
        X = a * X + (b * A + c * (A @ A)) @ X
    return X.t() if G.shape[0] > G.shape[1] else X


OPTIMIZERS = {"adam": FlatAdam, "muon": FlatMuon}


def make_optimizer(cfg, params, **kw):
    """The optimizer that cfg names (`optimizer: adam | muon`, adam when absent) on `params`."""
    name = getattr(cfg, "optimizer", "adam")
    if name not in OPTIMIZERS:
        raise ValueError("optimizer: %r is not one of %s" % (name, sorted(OPTIMIZERS)))
    return OPTIMIZERS[name](params, **kw)
