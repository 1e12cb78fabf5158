"""Fused optimizer / EMA step (SURVEY §8f "next" row 1): ``AdamW`` with torch.optim.AdamW's interface (param_groups, state_dict-free
stepping, per-group ``lr`` / ``weight_decay`` that a scheduler may rewrite every iteration — optim/adamw.py:16-46,
optim/scheduler/*) whose ``step()`` is ONE kernel launch over every parameter tensor (cvh_adamw_multi), optionally folding
``EMA.update_parameters`` (cvnets/misc/averaging_utils.py:43-55) into the same pass."""
from __future__ import annotations

import ctypes
import math
from typing import Iterable, List, Optional, Sequence, Tuple, Union

import torch
from torch.autograd import forward_ad

from . import _lib, ops
from .ops import _p, _stream


class AdamW(torch.optim.Optimizer):
    def __init__(self, params: Iterable, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
                 amsgrad: bool = False, ema: Optional[tuple] = None, ema_momentum: float = 0.0005):
        """ema = (model, ema_model): ema_model (a deepcopy of model, averaging_utils.py:33) is updated in the same pass"""
        if amsgrad:
            raise NotImplementedError("amsgrad is not on the HIP hot path")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        b = {tuple(g["betas"]) for g in self.param_groups} | {(g["eps"],) for g in self.param_groups}
        if len(b) != 2:
            raise NotImplementedError("per-group betas / eps are not supported (the reference uses one setting, optim/adamw.py:30-40)")
        self._plan = None
        self._loaded_state = {}
        self._rebuilds = 0
        self._ema = ema
        self.ema_momentum = float(ema_momentum)
        self._flat = None  # (flat fp32 buffer, [(parameter, view)]) when this optimizer owns the gradient storage (`flat_grads`)

    # ---- engine-driven use (cvnets_amd/launch.py): the reference's Trainer owns the loop, this object the gradient storage -------------
    @classmethod
    def from_torch(cls, optimizer: torch.optim.Optimizer, flat_grads: bool = True) -> "AdamW":
        """A fused AdamW with the parameter groups (parameters, lr, weight_decay, betas, eps — every other key rides along untouched, so a
        scheduler that rewrites ``param_groups[i]["lr"]`` keeps working) of a torch.optim.AdamW built by the reference's
        ``build_optimizer`` (optim/adamw.py:16-46).  State is not carried over: call it before the first step (or load a checkpoint after)."""
        if any(g.get("amsgrad", False) for g in optimizer.param_groups):
            raise NotImplementedError("amsgrad is not on the HIP hot path")
        groups = [{k: v for k, v in g.items()} for g in optimizer.param_groups]
        g0 = groups[0]
        new = cls(groups, lr=g0["lr"], betas=tuple(g0["betas"]), eps=g0["eps"], weight_decay=g0["weight_decay"])
        if flat_grads:
            new.adopt_flat_grads()
        return new

    def adopt_flat_grads(self) -> None:
        """Point every parameter's ``.grad`` into ONE flat fp32 buffer that this optimizer owns (parameters whose gradient already is a view
        of somebody's flat storage — cvnets_amd.ddp's buckets — are left alone).  ``zero_grad`` then is one memset whatever ``set_to_none``
        says, the gradient addresses never move (the one-launch plan stays valid), and with ``ops.set_inplace_param_grads(True)`` the
        backward kernels add straight into the buffer: no per-parameter AccumulateGrad work."""
        ps = [p for g in self.param_groups for p in g["params"] if p.requires_grad and p.grad is None and p.is_cuda and p.dtype == torch.float32]
        if not ps:
            return
        total = sum((p.numel() + 3) // 4 * 4 for p in ps)
        flat = torch.zeros(total, dtype=torch.float32, device=ps[0].device)
        views, off = [], 0
        for p in ps:
            v = flat[off: off + p.numel()].view_as(p)
            p.grad = v
            views.append((p, v))
            off += (p.numel() + 3) // 4 * 4
        self._flat = (flat, views)

    def zero_grad(self, set_to_none: bool = True) -> None:
        """torch's contract, except that gradients this optimizer owns are zeroed IN PLACE (engine/training_engine.py:224,307 passes
        set_to_none=True; dropping them would move every gradient address each iteration)."""
        if self._flat is None:
            return super().zero_grad(set_to_none=set_to_none)
        flat, views = self._flat
        owned = set()
        for p, v in views:
            owned.add(id(p))
            g = p.grad
            if g is None or g.data_ptr() != v.data_ptr():  # somebody replaced it (autograd allocates a fresh tensor for a None gradient)
                p.grad = v
        flat.zero_()
        for g in self.param_groups:
            for p in g["params"]:
                if id(p) not in owned and p.grad is not None:
                    if p.grad.grad_fn is not None:
                        p.grad.detach_()
                    p.grad.zero_()  # (e.g. views of cvnets_amd.ddp's buckets: stay in place as well)

    # -------------------------------------------------------------------------------------------------
    def _build(self):
        entries, skipped = [], []
        for gi, g in enumerate(self.param_groups):
            for p in g["params"]:
                if not p.requires_grad:
                    continue
                if p.grad is None:  # torch.optim.AdamW skips parameters without a gradient (no decay of weights or moments): so do we
                    skipped.append(p)
                else:
                    entries.append((p, gi))
        if not entries:
            raise RuntimeError("no parameter has a gradient")
        dev = entries[0][0].device
        if dev.type != "cuda":
            raise RuntimeError("cvnets_amd.optim.AdamW has no CPU path")
        ema_by_id = {}
        if self._ema is not None:  # pair parameters by registration order (EMA model = deepcopy of the model)
            model, ema_model = self._ema
            for p, e in zip(model.parameters(), ema_model.parameters()):
                if p.shape != e.shape:
                    raise RuntimeError("EMA model does not mirror the model")
                ema_by_id[id(p)] = e
        rows, offsets, off = [], [], 0
        for p, gi in entries:
            if p.dtype != torch.float32 or not p.is_contiguous():
                raise RuntimeError("parameters must be contiguous float32")
            e = ema_by_id.get(id(p))
            rows.append([p.data_ptr(), p.grad.data_ptr(), e.data_ptr() if e is not None else 0, off, p.numel(), gi, off, 0])
            offsets.append(off)
            off += (p.numel() + 3) // 4 * 4  # every tensor starts on a 4-element boundary: the kernel moves float4
        rows.append([0, 0, 0, 0, 0, 0, off, 0])
        plan = {
            "entries": entries, "skipped": skipped, "offsets": offsets, "total": off, "n": len(entries), "device": dev,
            "table": torch.tensor(rows, dtype=torch.int64, device=dev),
            "m": torch.zeros(off, dtype=torch.float32, device=dev), "v": torch.zeros(off, dtype=torch.float32, device=dev),
            "step": torch.zeros(1, dtype=torch.float32, device=dev),
            "hp": torch.zeros(len(self.param_groups), 2, dtype=torch.float32, device=dev),
            "hp_host": None, "grad_ptrs": [p.grad.data_ptr() for p, _ in entries],
        }
        old = self._plan
        if old is not None:  # gradients were re-allocated / the set of live parameters changed: carry the moments over per parameter
            prev = {id(p): o for (p, _), o in zip(old["entries"], old["offsets"])}
            for (p, _), o in zip(entries, offsets):
                po = prev.get(id(p))
                if po is not None:
                    plan["m"][o: o + p.numel()].copy_(old["m"][po: po + p.numel()])
                    plan["v"][o: o + p.numel()].copy_(old["v"][po: po + p.numel()])
            plan["step"] = old["step"]
            self._rebuilds += 1
            if self._rebuilds == 3:
                import warnings
                warnings.warn("cvnets_amd.optim.AdamW re-plans every step because the gradient tensors keep moving (zero_grad(set_to_none=True)?): "
                              "keep gradients in place (set_to_none=False or cvnets_amd.ddp's flat buckets) for the one-launch fast path")
        self._plan = plan
        self._apply_loaded_state()
        return plan

    def _valid(self, plan) -> bool:
        return all(p.grad is not None and p.grad.data_ptr() == gp for (p, _), gp in zip(plan["entries"], plan["grad_ptrs"])) \
            and all(p.grad is None for p in plan["skipped"])

    # ---- checkpointing: torch.optim.AdamW's state layout (step / exp_avg / exp_avg_sq per parameter index) -------------------------
    def _param_index(self):
        idx, i = {}, 0
        for g in self.param_groups:
            for p in g["params"]:
                idx[id(p)] = i
                i += 1
        return idx

    def state_dict(self):
        sd = super().state_dict()
        plan = self._plan
        if plan is not None:
            idx = self._param_index()
            step = plan["step"].detach().clone().reshape(())
            sd["state"] = {idx[id(p)]: {"step": step.clone(), "exp_avg": plan["m"][o: o + p.numel()].view_as(p).clone(),
                                        "exp_avg_sq": plan["v"][o: o + p.numel()].view_as(p).clone()}
                           for (p, _), o in zip(plan["entries"], plan["offsets"])}
        elif self._loaded_state:
            sd["state"] = self._loaded_state
        return sd

    def load_state_dict(self, state_dict):
        loaded = dict(state_dict.get("state", {}))
        super().load_state_dict({"state": {}, "param_groups": state_dict["param_groups"]})
        self._loaded_state = {int(k): v for k, v in loaded.items()}
        if self._plan is not None:
            self._apply_loaded_state()
            self._plan["hp_host"] = None  # the groups' lr / weight_decay may have changed

    def _apply_loaded_state(self):
        if not self._loaded_state or self._plan is None:
            return
        plan, idx = self._plan, self._param_index()
        steps = []
        for (p, _), o in zip(plan["entries"], plan["offsets"]):
            st = self._loaded_state.get(idx[id(p)])
            if st is None:
                continue
            plan["m"][o: o + p.numel()].copy_(st["exp_avg"].reshape(-1).to(plan["m"]))
            plan["v"][o: o + p.numel()].copy_(st["exp_avg_sq"].reshape(-1).to(plan["v"]))
            steps.append(float(st["step"]))
        if steps:
            plan["step"].fill_(max(steps))
        self._loaded_state = {}

    def sync_hyperparameters(self) -> None:
        """copy the per-group (lr, weight_decay) to the device table; call after a scheduler changed them (outside graph replay)."""
        plan = self._plan or self._build()
        host = [[float(g["lr"]), float(g["weight_decay"])] for g in self.param_groups]
        if host != plan["hp_host"]:
            plan["hp"].copy_(torch.tensor(host, dtype=torch.float32), non_blocking=True)  # plumbing: 2 floats per group
            plan["hp_host"] = host

    @torch.no_grad()
    def step(self, closure=None, inv_grad_scale: Optional[torch.Tensor] = None, sync_hyperparameters: bool = True):
        loss = closure() if closure is not None else None
        ops.finish_backward()  # side-stream dW work / deferred reductions of a backward whose end-of-backward callback was lost
        import sys
        _ddp = sys.modules.get(__package__ + ".ddp")
        if _ddp is not None:
            _ddp.exchange_pending()  # a hooked forward whose backward never reached the gradient exchange: run it before the update
        if not any(p.grad is not None for g in self.param_groups for p in g["params"]):
            return loss  # torch.optim.AdamW.step() with no gradients anywhere is a no-op
        plan = self._plan
        if plan is None or not self._valid(plan):
            plan = self._build()  # carries the moments of the previous plan over, parameter by parameter
        if sync_hyperparameters:
            self.sync_hyperparameters()
        g0 = self.param_groups[0]
        _lib.call("cvh_adamw_multi", _p(plan["table"]), plan["n"], plan["total"], _p(plan["m"]), _p(plan["v"]), _p(plan["hp"]),
                  float(g0["betas"][0]), float(g0["betas"][1]), float(g0["eps"]), _p(plan["step"]), _p(inv_grad_scale),
                  self.ema_momentum if self._ema is not None else 0.0, _stream())
        ops.invalidate_packed()  # parameters (and EMA parameters) changed through raw pointers: cached packed weights are stale
        return loss


class EMABuffers:
    """EMA of the model's floating-point BUFFERS (BatchNorm running statistics), the part of EMA.update_parameters that is not a
    parameter (averaging_utils.py:47-55 iterates the whole state_dict); integer buffers (num_batches_tracked) are copied."""

    def __init__(self, model: torch.nn.Module, ema_model: torch.nn.Module, momentum: float = 0.0005):
        rows, off, self.ints = [], 0, []
        for (k, s), (k2, d) in zip(model.named_buffers(), ema_model.named_buffers()):
            if k != k2 or s.shape != d.shape:
                raise RuntimeError("EMA model does not mirror the model's buffers")
            if s.dtype == torch.float32:
                rows.append([d.data_ptr(), s.data_ptr(), s.numel(), off])
                off += s.numel()
            else:
                self.ints.append((d, s))
        rows.append([0, 0, 0, off])
        self.n, self.total, self.momentum = len(rows) - 1, off, float(momentum)
        self.table = torch.tensor(rows, dtype=torch.int64, device=next(model.buffers()).device) if self.n else None
        self._keep = (model, ema_model)

    @torch.no_grad()
    def update(self):
        if self.n:
            _lib.call("cvh_lerp_multi", _p(self.table), self.n, self.total, self.momentum, _stream())
            ops.invalidate_packed()
        for d, s in self.ints:  # averaging an integer counter is a copy after the cast back (ema_v.copy_(...) on an int64 tensor)
            d.copy_((d * (1.0 - self.momentum) + self.momentum * s).to(d.dtype))


# ---- orthogonalised updates ------------------------------------------------------------------------------------------------------------
NS_COEFFICIENTS = (3.4445, -4.775, 2.0315)  # of the quintic step: maps singular values from (0, 1] towards 1, fastest growth at zero


def _check_ns(steps: int, coefficients: Sequence[float], eps: float) -> Tuple[int, float, float, float, float]:
    a, b, c = (float(x) for x in coefficients)
    if int(steps) < 1:
        raise ValueError(f"steps must be at least 1. Got: {steps}")
    if not abs(a) + abs(b) + abs(c) <= 15.0:
        raise ValueError(f"coefficients with |a| + |b| + |c| <= 15 are supported. Got: {tuple(coefficients)}")
    if not 0.0 <= eps < math.inf:
        raise ValueError(f"eps must not be negative. Got: {eps}")
    if not _lib.query("cvh_ns_bounded", int(steps), a, b, c):
        raise ValueError(f"coefficients whose steps let singular values grow beyond 15 in front of another step are not supported. Got: {tuple(coefficients)}, {steps} steps")
    return int(steps), a, b, c, float(eps)


def _check_matrix(rows: int, cols: int) -> None:
    if rows < 1 or cols < 1 or min(rows, cols) > 1 << 14 or max(rows, cols) > 1 << 20:
        raise NotImplementedError(f"matrices with a shorter side of 1 .. {1 << 14} and a longer one up to {1 << 20} are supported. Got: {rows} x {cols}")


def _by_cost(sizes: Sequence[Tuple[int, int]]) -> List[int]:
    """the longest products first: a launch over a list then ends with its short ones"""
    return sorted(range(len(sizes)), key=lambda i: -max(sizes[i]))


@torch.no_grad()
def orthogonalize(matrices: Union[torch.Tensor, Sequence[torch.Tensor]], steps: int = 5, coefficients: Sequence[float] = NS_COEFFICIENTS,
                  eps: float = 1e-7) -> Union[torch.Tensor, List[torch.Tensor]]:
    """Newton-Schulz orthogonalisation of matrices (one or a list of any shapes, all float32 or all bfloat16): x = u / (|u|_F + eps), then ``steps``
    times x <- (a I + b x x^T + c (x x^T)^2) x, the shorter side as rows.  The products are computed to float32 accuracy whatever the type
    of the matrices; the result has their type.  A list takes as many launches as one matrix.  A NaN or an infinity in a matrix makes its whole
    result NaN (and no other's).  Not differentiable: the result is detached.  Coefficients whose steps let singular values grow beyond 15 in front of another step are refused."""
    single = isinstance(matrices, torch.Tensor)
    mats = [matrices] if single else list(matrices)
    cfg = _check_ns(steps, coefficients, eps)
    for t in mats:
        if t.dim() != 2 or t.dtype not in (torch.float32, torch.bfloat16) or t.dtype != mats[0].dtype:
            raise RuntimeError(f"orthogonalize takes float32 or bfloat16 matrices of one dtype. Got: {t.dtype} {list(t.shape)}")
        _check_matrix(*t.shape)
    if getattr(forward_ad, "_current_level", 0) >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in mats):
        raise NotImplementedError("orthogonalize has no forward-mode derivatives")
    for t in mats:
        ops._check_dev(t)
        if t.device != mats[0].device:
            raise RuntimeError(f"the matrices must be on one device. Got: {t.device} and {mats[0].device}")
    if not mats:
        return []
    dev = mats[0].device
    src = [t.contiguous() for t in mats]
    out = [torch.empty_like(t) for t in src]
    table = (_lib.NsMatrix * len(src))(*[_lib.NsMatrix(_p(src[i]), _p(out[i]), None, None, *src[i].shape, 0, 1.0) for i in _by_cost([t.shape for t in src])])
    ws = torch.empty(_lib.query("cvh_ns_workspace_elems", ctypes.byref(table), len(src)), dtype=torch.float32, device=dev)
    ops.call_on(dev, "cvh_orthogonalize", ops._dt(src[0]), ctypes.byref(table), len(src), *cfg, _p(ws))
    return out[0] if single else out


def _capturing(device: torch.device) -> bool:
    return device.type == "cuda" and torch.cuda.is_current_stream_capturing()


class Muon(torch.optim.Optimizer):
    """Momentum whose update is orthogonalised, for the matrices of a model (dimensions behind the first are flattened, as in a convolution's
    [out, in, kh, kw]); vectors, embeddings and heads stay with ``AdamW``:

        mom <- momentum mom + grad;   u = grad + momentum mom (nesterov) or mom
        param <- (1 - lr weight_decay) param - lr max(1, rows / cols) ** 0.5 orthogonalize(u)

    ``param_groups`` with their own lr and weight_decay, which a scheduler may rewrite; ``state[p]["momentum_buffer"]`` and the usual state dict.
    One step is 2 + 3 ns_steps launches for up to 32 matrices.  Rates live on the device: a captured ``step(sync_hyperparameters=False)``
    follows ``sync_hyperparameters()`` calls between replays.  A step is captured after an eager one with the same parameters."""

    def __init__(self, params: Iterable, lr: float = 0.02, momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0, ns_steps: int = 5,
                 ns_coefficients: Sequence[float] = NS_COEFFICIENTS, eps: float = 1e-7):
        if not lr >= 0.0 or not weight_decay >= 0.0 or not 0.0 <= momentum < 1.0:
            raise ValueError(f"lr and weight_decay must not be negative, momentum in [0, 1). Got: {lr}, {weight_decay}, {momentum}")
        self._ns = _check_ns(ns_steps, ns_coefficients, eps)
        self._plan = None
        self._rates = []  # [device table of (lr, weight_decay) by group, its values], the newest last; a captured step goes on reading its own
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=bool(nesterov), weight_decay=weight_decay))

    def add_param_group(self, param_group) -> None:
        super().add_param_group(param_group)
        try:
            g, g0 = self.param_groups[-1], self.param_groups[0]
            if (g["momentum"], g["nesterov"]) != (g0["momentum"], g0["nesterov"]):
                raise NotImplementedError("per-group momentum / nesterov are not supported")
            for p in g["params"]:
                if p.dim() < 2:
                    raise ValueError(f"Muon takes matrices (two or more dimensions); give vectors to AdamW. Got: {list(p.shape)}")
                if p.dtype != torch.float32 or not p.is_contiguous():
                    raise RuntimeError("parameters must be contiguous float32")
                _check_matrix(p.shape[0], p.numel() // max(1, p.shape[0]))
        except Exception:
            self.param_groups.pop()
            raise

    @torch.no_grad()
    def load_state_dict(self, state_dict) -> None:
        """into the momentum that is there (zeros where none is loaded): a captured step goes on reading and writing it"""
        held = {p: s["momentum_buffer"] for p, s in self.state.items() if "momentum_buffer" in s}
        super().load_state_dict(state_dict)
        for p, buf in held.items():
            new = self.state[p].get("momentum_buffer")
            if new is None or new.shape == buf.shape:
                self.state[p]["momentum_buffer"] = buf.zero_() if new is None else buf.copy_(new)

    def _entries(self):
        out = []
        for gi, g in enumerate(self.param_groups):
            for p in g["params"]:
                if p.grad is not None:
                    if p.grad.is_sparse or p.grad.dtype != torch.float32:
                        raise RuntimeError("gradients must be dense float32")
                    out.append((p, p.grad if p.grad.is_contiguous() else p.grad.contiguous(), gi))
        return out

    def _build(self, entries):
        dev = entries[0][0].device
        for p, _, _ in entries:
            ops._check_dev(p)
            if p.device != dev:
                raise RuntimeError(f"the parameters must be on one device. Got: {p.device} and {dev}")
            buf = self.state[p].get("momentum_buffer")
            if not p.is_contiguous() or (buf is not None and buf.shape != p.shape):
                raise RuntimeError(f"a parameter became another matrix: {list(p.shape)}, contiguous {p.is_contiguous()}, its momentum {None if buf is None else list(buf.shape)}")
            _check_matrix(p.shape[0], p.numel() // max(1, p.shape[0]))
            if buf is None or buf.dtype != torch.float32 or not buf.is_contiguous() or buf.device != dev:  # (a loaded state may be another type's)
                if _capturing(dev):  # every replay would make it again
                    raise RuntimeError("a captured step needs the momentum of its parameters: take an eager step with them before the capture")
                self.state[p]["momentum_buffer"] = torch.zeros_like(p) if buf is None else buf.to(device=dev, dtype=torch.float32).contiguous()
        sizes = [(p.shape[0], p.numel() // p.shape[0]) for p, _, _ in entries]
        rows = [_lib.NsMatrix(src=_p(entries[i][1]), momentum=_p(self.state[entries[i][0]]["momentum_buffer"]), param=_p(entries[i][0]), rows=sizes[i][0],
                              cols=sizes[i][1], group=entries[i][2], gain=math.sqrt(max(1.0, sizes[i][0] / sizes[i][1]))) for i in _by_cost(sizes)]
        table = (_lib.NsMatrix * len(rows))(*rows)
        self._plan = {"table": table, "n": len(rows), "need": _lib.query("cvh_ns_workspace_elems", ctypes.byref(table), len(rows)), "key": self._key(entries)}
        return self._plan

    def _key(self, entries):
        """what the plan holds: addresses, and the layouts that stand behind them (a square matrix's transposed view has its address and shape)"""
        bufs = [self.state[p].get("momentum_buffer") for p, _, _ in entries]
        return [(p.data_ptr(), p.shape, p.stride(), g.data_ptr(), gi, None if m is None else (m.data_ptr(), m.shape, m.stride(), m.dtype)) for (p, g, gi), m in zip(entries, bufs)]

    def _has_rates(self, device) -> bool:
        """whether the newest table has a row for every group (the kernels read it), where the parameters are"""
        return bool(self._rates) and len(self._rates[-1][0]) >= len(self.param_groups) and self._rates[-1][0].device == device

    def sync_hyperparameters(self) -> None:
        """copy the groups' (lr, weight_decay) to the device tables; call after a scheduler changed them (outside graph replay)"""
        host = [[float(g["lr"]), float(g["weight_decay"])] for g in self.param_groups]
        device = next(p.device for g in self.param_groups for p in g["params"])
        if _capturing(device):  # what is copied to the device comes from a temporary of the host's
            if not self._has_rates(device) or any(values != host[:len(table)] for table, values in self._rates):
                raise RuntimeError("the groups' rates changed: call sync_hyperparameters() before the capture, not in it")
            return
        if not self._has_rates(device):
            self._rates.append([torch.zeros(len(host), 2, dtype=torch.float32, device=device), None])
        for entry in self._rates:
            table, values = entry[0], host[:len(entry[0])]
            if values != entry[1]:
                table[:len(values)].copy_(torch.tensor(values, dtype=torch.float32), non_blocking=True)  # plumbing: 2 floats per group
                entry[1] = values

    @torch.no_grad()
    def step(self, closure=None, sync_hyperparameters: bool = True):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        ops.finish_backward()
        import sys
        _ddp = sys.modules.get(__package__ + ".ddp")
        if _ddp is not None:
            _ddp.exchange_pending()
        entries = self._entries()
        if not entries:
            return loss
        dev = entries[0][0].device
        ops._check_dev(entries[0][0])
        plan = self._plan
        if plan is None or plan["key"] != self._key(entries):
            plan = self._build(entries)
        if sync_hyperparameters or not self._has_rates(dev):
            self.sync_hyperparameters()
        g0 = self.param_groups[0]
        for g in self.param_groups:  # (they may be rewritten, or loaded)
            if (g["momentum"], g["nesterov"]) != (g0["momentum"], g0["nesterov"]):
                raise NotImplementedError("per-group momentum / nesterov are not supported")
        # a workspace of this step's own, on its stream: a graph takes one from its own memory, so that two of them may be replayed side by side
        ws = torch.empty(plan["need"], dtype=torch.float32, device=dev)
        ops.call_on(dev, "cvh_muon_step", ctypes.byref(plan["table"]), plan["n"], *self._ns, float(g0["momentum"]), int(g0["nesterov"]), _p(self._rates[-1][0]), _p(ws))
        ops.invalidate_packed()
        return loss
