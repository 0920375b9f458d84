"""AdamW on the HIP multi-tensor kernel (csrc/adamw.hip) -- SURVEY.md 8(f) rank 1.  Same update rule, hyper-parameters,
param-group handling and state-dict layout (`step`, `exp_avg`, `exp_avg_sq`, one `step` per tensor) as torch.optim.AdamW
(which the reference gets from timm's create_optimizer_v2, train.py:662), one launch per parameter group instead of a
chain of foreach kernels, and the CGA weight freeze (cga.py:953-1013) folded into the same pass via `set_frozen`.

hipGraph: a captured launch keeps its arguments, so inside a capture (engine.GraphedTrainStep) step() launches the
`_dev` form of the kernel, which reads lr and the bias corrections from device memory, and leaves the step counters
alone; `advance_for_replay()` -- called before every replay -- advances the counters on the host and stores the new
scalars (formed by the same host arithmetic as the eager path: bit-identical updates)."""
import functools
import math

import numpy as np
import torch

from . import ops


class _GraphClass:
    """Parameters of one group that have taken the same number of steps: one captured launch, one device scalar block."""
    __slots__ = ("group", "params", "hyper", "fixed")

    def __init__(self, group, params, hyper):
        self.group, self.params, self.hyper = group, params, hyper
        self.fixed = None            # settings that the captured launches hold by value (FusedMuon)


class FusedAdamW(torch.optim.Optimizer):
    MAX_GRAPH_CLASSES = 32

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2):
        if lr < 0 or eps < 0 or not 0 <= betas[0] < 1 or not 0 <= betas[1] < 1 or weight_decay < 0:
            raise ValueError("FusedAdamW: invalid hyper-parameter")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        self._frozen = {}            # id(param) -> {0,1} fp32 mask of the parameter's shape (CGA), or absent
        self._graph_classes = None   # list of _GraphClass while / after a capture
        self._hyper_pool = None

    def set_frozen(self, param, mask):
        """CGA: elements with mask != 0 take no update this step (gradient masked, weight restored)."""
        if mask is None:
            self._frozen.pop(id(param), None)
        else:
            self._frozen[id(param)] = mask

    def clear_frozen(self):
        self._frozen.clear()

    def _table(self, plist):
        """Host array of {p, g, m, v, frozen, n} (the kernel launch copies it into its arguments: nothing goes to the
        device ahead of the launch, so fresh gradient tensors every step cost nothing)."""
        tens = np.empty((len(plist), 6), dtype=np.int64)
        for i, p in enumerate(plist):
            st = self.state[p]
            f = self._frozen.get(id(p))
            tens[i] = (p.data_ptr(), p.grad.data_ptr(), st["exp_avg"].data_ptr(), st["exp_avg_sq"].data_ptr(),
                       0 if f is None else f.data_ptr(), p.numel())
        return tens

    def _ready(self, group):
        """Parameters of the group that take part in this step (have a gradient), state created on first use."""
        plist = [p for p in group["params"] if p.grad is not None]
        for p in plist:
            if not p.is_cuda or p.dtype != torch.float32 or not p.is_contiguous() or not p.grad.is_contiguous():
                raise RuntimeError("FusedAdamW: contiguous fp32 parameters on a HIP device only (no CPU fallback)")
            st = self.state[p]
            if not st:
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("FusedAdamW: optimizer state must exist before a capture (moments allocated inside a "
                                       "capture would be re-zeroed by every replay); run an eager step first")
                st["step"] = torch.tensor(0.0)
                st["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
        return plist

    def _classes(self, plist):
        """Split by the number of steps taken so far: torch keeps one `step` per tensor, and a parameter that skipped a
        step (no gradient) must get its own bias corrections.  Normally one class."""
        out, seen = {}, {}
        for p in plist:
            st = self.state[p]["step"]
            t = seen.get(id(st))
            if t is None:
                t = seen[id(st)] = int(st.item() if torch.is_tensor(st) else st)
            out.setdefault(t, []).append(p)
        return out

    def _set_step(self, ps, t):
        """state['step'] = t for every parameter of the class.  The tensors of a class share ONE cpu tensor object (150
        fresh tensors per step cost more host time than the launch); it is split when the class splits."""
        first = self.state[ps[0]]["step"]
        shared = torch.is_tensor(first) and all(self.state[p]["step"] is first for p in ps)
        if shared:
            users = sum(1 for g in self.param_groups for p in g["params"] if self.state.get(p, {}).get("step") is first)
            shared = users == len(ps)
        if shared:
            first.fill_(float(t))
        else:
            obj = torch.tensor(float(t))
            for p in ps:
                self.state[p]["step"] = obj

    @staticmethod
    def _hyper(group, t):
        b1, b2 = group["betas"]
        h = np.empty(8, dtype=np.float32)
        ops._chk(ops.lib().ofq_adamw_hyper_pack(h.ctypes.data, float(group["lr"]), float(b1), float(b2), float(group["eps"]),
                                                float(group["weight_decay"]), 1.0 - b1 ** t, 1.0 - b2 ** t),
                 "ofq_adamw_hyper_pack")
        return h

    # ---------------------------------------------------------------------------------------------- hipGraph
    def begin_capture(self, device):
        self._graph_classes = []
        self._hyper_pool = torch.zeros(self.MAX_GRAPH_CLASSES * 8, dtype=torch.float32, device=device)

    def _advance_class(self, gc):
        """One replayed step of a captured class: its step counter, and the eight scalars that its launch reads."""
        t = int(self.state[gc.params[0]]["step"].item()) + 1
        self._set_step(gc.params, t)
        return self._hyper(gc.group, t)

    def advance_for_replay(self):
        """Before every replay of a graph that holds this optimizer's step: advance the step counters of the captured
        classes and store their scalars (lr, bias corrections ...) where the captured launches read them."""
        if not self._graph_classes:
            raise RuntimeError("FusedAdamW.advance_for_replay: no captured step")
        vals = np.empty(len(self._graph_classes) * 8, dtype=np.float32)
        for i, gc in enumerate(self._graph_classes):
            vals[8 * i:8 * i + 8] = self._advance_class(gc)
        lib, stream = ops.lib(), ops._stream()
        for off in range(0, vals.size, 32):
            chunk = np.ascontiguousarray(vals[off:off + 32])
            ops._chk(lib.ofq_store_f32(self._hyper_pool.data_ptr() + 4 * off, chunk.ctypes.data, int(chunk.size), stream),
                     "ofq_store_f32")

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        assert ops.lib().ofq_adamw_tensor_entry_bytes() == 48
        capturing = torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing()
        if capturing and self._graph_classes is None:
            raise RuntimeError("%s.step inside a stream capture needs begin_capture() first (engine.GraphedTrainStep)"
                               % type(self).__name__)
        for group in self.param_groups:
            self._step_group(group, capturing)
        return loss

    def _captured_hyper(self, group, ps):
        """The eight device scalars of a launch that is being captured, refreshed by advance_for_replay()."""
        i = len(self._graph_classes)
        if i >= self.MAX_GRAPH_CLASSES:
            raise RuntimeError("%s: more than %d (group, step) classes in one captured step" % (type(self).__name__, i))
        hyper = self._hyper_pool[8 * i:8 * i + 8]
        self._graph_classes.append(_GraphClass(group, ps, hyper))
        return hyper

    def _step_group(self, group, capturing):
        plist = self._ready(group)
        if not plist:
            return
        lib = ops.lib()
        for t0, ps in self._classes(plist).items():
            tens = self._table(ps)
            # the device's step-guard word (engine's step writes it between the collectives and this call; None before the
            # first such step): while it is non-zero the launch updates nothing -- see ops.step_guard
            guard = ops.step_guard_ptr(ps[0].device) or None
            if capturing:
                hyper = self._captured_hyper(group, ps)
                ops._chk(lib.ofq_adamw_multi_dev_g(tens.ctypes.data, len(ps), hyper.data_ptr(), guard, ops._stream()),
                         "ofq_adamw_multi_dev_g")
                continue
            t = t0 + 1
            self._set_step(ps, t)
            b1, b2 = group["betas"]
            ops._chk(lib.ofq_adamw_multi_g(tens.ctypes.data, len(ps), float(group["lr"]), float(b1), float(b2),
                                           float(group["eps"]), float(group["weight_decay"]), 1.0 - b1 ** t, 1.0 - b2 ** t,
                                           guard, ops._stream()), "ofq_adamw_multi_g")


# ------------------------------------------------------------------------------------------------------ Newton-Schulz
NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)


@functools.lru_cache(maxsize=64)
def _newton_schulz_in_range(coefficients, steps):
    """The kernels hold X, X X^T and b A + c A A as 16-bit planes of the value times 2^10: coefficients that drive a singular value
    (they all start in [0, 1]) or an eigenvalue of the polynomial past what the planes hold are refused."""
    a, b, c = coefficients
    x = np.linspace(0.0, 1.0, 4097)
    with np.errstate(over="ignore", invalid="ignore"):
        for _ in range(steps):
            p = b * x * x + c * x ** 4
            if not (np.abs(p).max() < 32 and (x * x).max() < 32):
                return False
            x = a * x + p * x
    return bool(np.abs(x).max() < 32)


def _check_newton_schulz(who, coefficients, steps, eps):
    if not isinstance(steps, int) or not 0 <= steps <= 100:
        raise ValueError("%s: the number of steps must be an integer from 0 to 100 (got %r)" % (who, steps))
    if len(coefficients) != 3 or not all(math.isfinite(c) for c in coefficients):
        raise ValueError("%s: three finite coefficients (got %r)" % (who, coefficients))
    if not eps > 0:
        raise ValueError("%s: eps must be positive (got %r)" % (who, eps))
    if not _newton_schulz_in_range(tuple(float(c) for c in coefficients), steps):
        raise ValueError("%s: these coefficients let the singular values grow out of range: %r" % (who, tuple(coefficients)))


@torch.no_grad()
def orthogonalize(matrices, steps=5, coefficients=NS_COEFFICIENTS, eps=1e-7):
    """Newton-Schulz orthogonalisation of a matrix, or of each of a list of matrices in the same launches (csrc/newton_schulz.hip):
    X = G / max(|G|_F, eps), then `steps` times X <- a X + (b A + c A A) X with A = X X^T.  fp32 or bf16 (each result in its
    matrix's type); the chain itself has fp32's precision for both.  A zero matrix stays zero."""
    single = torch.is_tensor(matrices)
    mats = [matrices] if single else list(matrices)
    _check_newton_schulz("orthogonalize", coefficients, steps, eps)
    for g in mats:
        if g.dim() != 2:
            raise ValueError("orthogonalize: matrices only (got shape %s)" % (tuple(g.shape),))
        if not g.is_cuda or g.dtype not in (torch.float32, torch.bfloat16):
            raise RuntimeError("ofq_amd: orthogonalize: float32 or bfloat16 matrices on a HIP device (got %s on %s); there is no CPU "
                               "fallback" % (g.dtype, g.device))
    outs = [torch.empty(g.shape, dtype=g.dtype, device=g.device) for g in mats]
    runs = {}
    for g, o in zip(mats, outs):
        if g.numel():
            runs.setdefault((g.device, g.dtype), []).append((g.contiguous(), o))
    for (dev, dtype), pairs in runs.items():
        table = np.array([(g.data_ptr(), 0, o.data_ptr(), g.shape[0], g.shape[1], 1.0, 0.0) for g, o in pairs], dtype=ops.NS_ENTRY)
        with ops.on_device(dev):
            ops.newton_schulz(table, dtype == torch.bfloat16, steps, coefficients, eps, device=dev)
    return outs[0] if single else outs


class FusedMuon(FusedAdamW):
    """Momentum with an orthogonalised update for the matrices of a model, with torch.optim.Muon's rule and argument names:
        m <- m + (1 - momentum)(g - m);  u = g + momentum (m - g) (nesterov) or m;  O = orthogonalize(u)
        p <- p (1 - lr weight_decay) - lr s O
    s = sqrt(max(1, rows / columns)) (adjust_lr_fn None or "original") or 0.2 sqrt(max(rows, columns)) ("match_rms_adamw": an update of
    AdamW's size, so that both rules take the same lr).  All matrices of a group go through the same launches.
    A group with use_muon=False is updated by FusedAdamW's rule (betas, adamw_eps): embeddings, heads, vectors.  Parameters are
    contiguous fp32 on a HIP device; Muon groups hold matrices only.  Captured steps work as FusedAdamW's do: a Muon group's follow lr and
    weight_decay, and refuse a replay after a change of its other settings."""

    def __init__(self, params, lr=1e-3, weight_decay=0.1, momentum=0.95, nesterov=True, ns_coefficients=NS_COEFFICIENTS, eps=1e-7,
                 ns_steps=5, adjust_lr_fn=None, betas=(0.9, 0.999), adamw_eps=1e-8):
        if lr < 0 or weight_decay < 0 or not 0 <= momentum < 1 or adamw_eps < 0 or not 0 <= betas[0] < 1 or not 0 <= betas[1] < 1:
            raise ValueError("FusedMuon: invalid hyper-parameter")
        torch.optim.Optimizer.__init__(self, params, dict(
            lr=lr, weight_decay=weight_decay, momentum=momentum, nesterov=nesterov, ns_coefficients=tuple(ns_coefficients), eps=eps,
            ns_steps=ns_steps, adjust_lr_fn=adjust_lr_fn, use_muon=True, betas=betas, adamw_eps=adamw_eps))
        self._frozen = {}
        self._graph_classes = None
        self._hyper_pool = None

    def add_param_group(self, group):
        super().add_param_group(group)
        group = self.param_groups[-1]
        try:
            if not group["use_muon"]:
                return
            _check_newton_schulz("FusedMuon", group["ns_coefficients"], group["ns_steps"], group["eps"])
            if group["adjust_lr_fn"] not in (None, "original", "match_rms_adamw"):
                raise ValueError("FusedMuon: adjust_lr_fn must be None, 'original' or 'match_rms_adamw' (got %r)"
                                 % (group["adjust_lr_fn"],))
            if len({id(p) for p in group["params"]}) != len(group["params"]):
                raise ValueError("FusedMuon: a parameter is in its group twice")
            for p in group["params"]:
                if p.dim() != 2:
                    raise ValueError("FusedMuon: matrices only in a Muon group (got shape %s); give other parameters a group with "
                                     "use_muon=False" % (tuple(p.shape),))
        except ValueError:
            self.param_groups.pop()
            raise

    def set_frozen(self, param, mask):
        if mask is not None and any(p is param for g in self.param_groups if g["use_muon"] for p in g["params"]):
            raise RuntimeError("FusedMuon: an orthogonalised update cannot leave single elements out (CGA's weight freeze): give the "
                               "parameter a group with use_muon=False")
        super().set_frozen(param, mask)

    @staticmethod
    def _lr_scale(group, shape):
        r, c = shape
        return 0.2 * math.sqrt(max(r, c)) if group["adjust_lr_fn"] == "match_rms_adamw" else math.sqrt(max(1.0, r / c))

    _FIXED = ("momentum", "nesterov", "ns_coefficients", "eps", "ns_steps", "adjust_lr_fn")

    def _capture_muon(self, group):
        """The device scalars of a captured Muon group's launches; everything else they hold by value."""
        hyper = self._captured_hyper(group, None)
        self._graph_classes[-1].fixed = [group[k] for k in self._FIXED]
        return hyper

    def advance_for_replay(self):
        for gc in self._graph_classes or ():
            if gc.fixed is not None and gc.fixed != [gc.group[k] for k in self._FIXED]:
                raise RuntimeError("FusedMuon: a captured step follows lr and weight_decay; %s changed since: capture the step again"
                                   % ", ".join(k for k, old in zip(self._FIXED, gc.fixed) if gc.group[k] != old))
        super().advance_for_replay()

    def _advance_class(self, gc):
        if not gc.group["use_muon"]:
            return super()._advance_class(gc)
        h = np.zeros(8, dtype=np.float32)
        h[0] = gc.group["lr"]
        h[1] = np.float32(1) - np.float32(gc.group["lr"]) * np.float32(gc.group["weight_decay"])      # as the by-value launch forms it
        return h

    def _step_group(self, group, capturing):
        if not group["use_muon"]:
            return super()._step_group(_AdamWView(group), capturing)
        runs, scales, state, f32 = {}, {}, self.state, torch.float32
        for p in group["params"]:
            g = p.grad
            if g is None or p.numel() == 0:
                continue
            dev = p.device
            if dev.type != "cuda" or p.dtype != f32 or not p.is_contiguous() or g.dtype != f32 or not g.is_contiguous() or g.device != dev:
                raise RuntimeError("FusedMuon: contiguous fp32 parameters and gradients on a HIP device only (no CPU fallback)")
            shape = p.shape
            buf = state[p].get("momentum_buffer")
            if buf is None:
                if capturing:
                    raise RuntimeError("FusedMuon: optimizer state must exist before a capture (a buffer allocated inside a capture "
                                       "would be re-zeroed by every replay); run an eager step first")
                buf = state[p]["momentum_buffer"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
            elif buf.dtype != f32 or buf.shape != shape or not buf.is_contiguous() or buf.device != dev:
                raise RuntimeError("FusedMuon: momentum_buffer must be a contiguous fp32 tensor of its parameter's shape and device")
            scale = scales.get(shape)
            if scale is None:
                scale = scales[shape] = self._lr_scale(group, shape)
            rows = runs.get(dev)
            if rows is None:
                rows = runs[dev] = []
            rows.append((g.data_ptr(), buf.data_ptr(), p.data_ptr(), shape[0], shape[1], scale, 0.0))
        for dev, rows in runs.items():
            hyper = self._capture_muon(group).data_ptr() if capturing else None
            with ops.on_device(dev):
                ops.newton_schulz(np.array(rows, dtype=ops.NS_ENTRY), False, group["ns_steps"], group["ns_coefficients"], group["eps"],
                                  float(group["lr"]), float(group["weight_decay"]), float(group["momentum"]), group["nesterov"], hyper,
                                  ops.step_guard_ptr(dev) or None, device=dev)


class _AdamWView(dict):
    """A Muon optimiser's AdamW group as FusedAdamW reads it: eps is its adamw_eps, everything else the live group's (a captured class keeps
    this view, and the scheduler changes the group's lr)."""

    def __init__(self, group):
        super().__init__()
        self._group = group

    def __getitem__(self, key):
        return self._group["adamw_eps" if key == "eps" else key]
