"""Adam on the HIP kernel (ps_adam_step), torch.optim.Adam-compatible numerics for the reference's settings
(ns/engine/optimizers.py:73-170: one Adam per parameter group, lr 1e-2, eps 1e-15, weight_decay 1e-5); and for weight matrices, single or
stacked by expert, the orthogonalised update (newton_schulz) and the momentum step that applies it (HipMuon)."""
from __future__ import annotations

import functools
import math
from typing import Iterable, List, Optional, Sequence, Tuple

import ctypes

import torch

from ._lib import check, lib
from .dist import flat_grads_of, intersect_ranges
from .experts import DTYPE_CODES, _gpu, _on, _typed
from .ops import _p, _stream, join_side_streams


class HipAdam:
    def __init__(self, params: Iterable[torch.nn.Parameter], lr: float = 1e-2, betas=(0.9, 0.999), eps: float = 1e-15,
                 weight_decay: float = 1e-5, flat_grads=None, grad_scale: float = 1.0):
        """grad_scale: factor applied to every gradient inside the kernel before the weight decay is added.  1.0 (default) =
        the reference's default path: with update_grad_scaler=False its Trainer calls optimizer.step() on the gradients exactly
        as backward left them, loss scale included (ns/engine/trainer.py:481-486, optimizers.py:133-140).  1 / loss_scale = its
        update_grad_scaler=True branch, where GradScaler.step unscales first (optimizers.py:118-131).
        flat_grads: a presight_amd.dist.FlatGrads over exactly `params` -> parameters and both moments are moved into
        flat buffers of the same layout (every parameter's storage is re-pointed to a view of the flat buffer, values
        kept) and the whole update is ONE kernel launch over the flat range instead of one per tensor."""
        self.params: List[torch.nn.Parameter] = [p for p in params if p.requires_grad and p.numel() > 0]
        for p in self.params:
            if not p.is_cuda or p.dtype != torch.float32 or not p.is_contiguous():
                raise RuntimeError("HipAdam: parameters must be contiguous fp32 CUDA tensors")
        self.lr, self.betas, self.eps, self.weight_decay = lr, betas, eps, weight_decay
        self.grad_scale = float(grad_scale)
        self.fused_armed = False  # enable_fused_tables: only a backward pass the trainer has armed applies the tables' update
        self.step_count = 0  # optimizer steps taken (informational; the bias corrections use the per-parameter counts)
        self.steps: List[int] = [0] * len(self.params)  # torch's state[p]["step"]
        self.flat = None
        if flat_grads is not None:
            if len(flat_grads.params) != len(self.params) or any(a is not b for a, b in zip(flat_grads.params, self.params)):
                raise ValueError("HipAdam: flat_grads must cover exactly the optimizer's parameters, in the same order")
            dev = self.params[0].device
            fp = torch.zeros(flat_grads.total, device=dev, dtype=torch.float32)  # padding stays 0 (grad 0, decay of 0)
            fm, fv = torch.zeros_like(fp), torch.zeros_like(fp)
            self.exp_avg, self.exp_avg_sq = [], []
            with torch.no_grad():
                for p, off in zip(self.params, flat_grads.offsets):
                    n = p.numel()
                    view = fp[off:off + n].view_as(p)
                    view.copy_(p.data)
                    p.data = view
                    self.exp_avg.append(fm[off:off + n].view_as(p))
                    self.exp_avg_sq.append(fv[off:off + n].view_as(p))
            self.flat = (fp, flat_grads.flat, fm, fv)
            self.flat_grads = flat_grads
        else:
            self.exp_avg = [torch.zeros_like(p) for p in self.params]
            self.exp_avg_sq = [torch.zeros_like(p) for p in self.params]

    # ------------------------------------------------------------------ Adam inside the table backward (single-process training)
    def enable_fused_tables(self, indices: Sequence[int]) -> None:
        """The hash tables self.params[i], i in indices, are updated INSIDE their table backward (ps_grid_scatter_binned_adam: the
        accumulate pass applies this optimizer's element update to every slice it finishes, the gradient never reaches memory) instead
        of by step().  Valid when nobody needs the gradient itself: no exchange (one process / one tile per GPU), no found-inf check
        (update_grad_scaler=False), and one gradient contribution per table and step (a second one raises).  Same bits as step():
        both run csrc/adam_core.hpp::adam_update on the same fp32 gradient."""
        if self.flat is None:
            raise RuntimeError("HipAdam.enable_fused_tables: needs the flat buffers (flat_grads=...)")
        for i in indices:
            p = self.params[i]
            p._ps_fused_adam, p._ps_fused_index, p._ps_fused_done = self, i, False

    def disable_fused_tables(self) -> None:
        for p in self.params:
            if getattr(p, "_ps_fused_adam", None) is self:
                p._ps_fused_adam = None

    def fused_table_args(self, tables: Sequence[torch.nn.Parameter], routed: bool):
        """Called by the table backward (field_ops._scatter / _ms_scatter) right before its launch: -> the Adam arguments of
        ps_grid_scatter_binned_adam (routed: of ps_grid_scatter_binned_ms_adam) for THIS step's update of `tables`, or None when it has
        to go through step() after all.  Advances the host-side step counts and marks the tables as updated: step() skips them and
        FlatGrads.zero_ leaves their (still zero) gradient ranges alone."""
        if not self.fused_armed:
            return None  # a backward pass outside Trainer.step (gradient inspection, tests): plain gradients, step() does the update
        fg = self.flat_grads
        for t in tables:
            if getattr(t, "_ps_fused_done", False):
                raise RuntimeError("presight_amd: a hash table whose Adam update is fused into its backward received a second gradient "
                                   "contribution in one step (HipAdam.enable_fused_tables needs exactly one)")
        gids = [getattr(t, "_ps_group", None) if fg.n_groups else None for t in tables]
        if not routed and gids[0] is not None:
            return None  # a routed sub-field called on its own: whether it counts as updated is the device's decision
        idx = [t._ps_fused_index for t in tables]
        host = [i for i, g_ in zip(idx, gids) if g_ is None]
        if host and len({self.steps[i] for i in host}) != 1:
            return None
        step = self.steps[host[0]] + 1 if host else 0
        for i in host:
            self.steps[i] += 1
        for t in tables:
            t._ps_fused_done = True
        fp, fgr, fm, fv = self.flat
        args = (_p(fgr), _p(fp), _p(fm), _p(fv), self.lr, self.betas[0], self.betas[1], self.eps, self.weight_decay, self.grad_scale, step)
        if not routed:
            return args
        if all(g_ is None for g_ in gids):
            return args + (None, None, None)
        key = tuple(-1 if g_ is None else g_ for g_ in gids)
        tbl = self._fused_gid_tables.get(key) if hasattr(self, "_fused_gid_tables") else None
        if tbl is None:
            if not hasattr(self, "_fused_gid_tables"):
                self._fused_gid_tables = {}
            tbl = torch.tensor(key, dtype=torch.int32, device=fp.device)
            self._fused_gid_tables[key] = tbl
        return args + (_p(tbl), _p(fg.group_flags), _p(fg.group_steps))

    @torch.no_grad()
    def step(self, skip=(), subset=None):
        """skip: indices of parameters whose update is withheld this step although they received a gradient (GradScaler.step
        found an inf / nan in their group): treated like parameters without a gradient.
        subset: only these parameter indices are updated by this call (the step is issued in pieces: presight_amd.trainer.Trainer
        runs the fields' piece on a second stream underneath the next step's proposal sampling); launches go to the current stream.
        torch.optim.Adam semantics per PARAMETER: state["step"] (the bias-correction exponent) advances only for parameters
        that received a gradient this step; the others are skipped entirely (no decay, no moment update), like torch with
        grad None after zero_grad(set_to_none=True).  Proposal networks (a gradient every ~6th step after warm-up) and
        sub-fields that saw no sample therefore keep their own, smaller step counts."""
        if subset is None or 0 in subset or not self.params:
            self.step_count += 1  # (a step issued in pieces counts once: with the piece that holds parameter 0)
        s = _stream()
        if self.flat is not None:
            fg = self.flat_grads
            fg._join_side_streams()
            idx = [i for i in fg.touched_params() if i not in skip and (subset is None or i in subset)
                   and not getattr(self.params[i], "_ps_fused_done", False)]  # (updated inside their table backward already)
            if skip and fg.n_groups:  # device-decided groups of withheld parameters: lower their flags
                for g_ in {getattr(self.params[i], "_ps_group", None) for i in skip} - {None}:
                    fg.group_flags[g_] = 0
            gid = [getattr(self.params[i], "_ps_group", None) if fg.n_groups else None for i in idx]
            for i, gr in zip(idx, gid):
                if gr is None:
                    self.steps[i] += 1  # (the step counts of device-decided groups live on the device: fg.group_steps)
            # adjacent touched parameters of the same group / with the same host step count merge into one range; in sharded
            # data-parallel mode this rank only updates the shard it owns (reduce-scatter -> Adam on the shard -> all-gather)
            runs: List[list] = []
            for i, gr in zip(idx, gid):
                a, b = fg.offsets[i], fg.offsets[i] + fg._pad(self.params[i].numel())
                key = ("g", gr) if gr is not None else ("s", self.steps[i])
                if runs and runs[-1][1] == a and runs[-1][2] == key:
                    runs[-1][1] = b
                else:
                    runs.append([a, b, key])
            owned = fg.owned_ranges()
            ranges = []
            for a, b, key in runs:
                for x, y in intersect_ranges([(a, b)], owned):
                    ranges.append((x, y - x, key))
            if ranges:
                n = len(ranges)
                starts = (ctypes.c_int64 * n)(*[r[0] for r in ranges])
                counts = (ctypes.c_int64 * n)(*[r[1] for r in ranges])
                steps = (ctypes.c_int * n)(*[(r[2][1] if r[2][0] == "s" else 0) for r in ranges])
                groups = (ctypes.c_int * n)(*[(r[2][1] if r[2][0] == "g" else -1) for r in ranges])
                check(lib().ps_adam_step_ranges(_p(self.flat[0]), _p(self.flat[1]), _p(self.flat[2]), _p(self.flat[3]), n, starts, counts,
                                                steps, groups, _p(fg.group_flags), _p(fg.group_steps), fg.n_groups, self.lr,
                                                self.betas[0], self.betas[1], self.eps, self.weight_decay, self.grad_scale, s),
                      "ps_adam_step_ranges")
            fg.gather_params(self.flat[0], [(a, b) for a, b, _ in runs])  # no-op unless the exchange is sharded
            return
        for i, (p, m, v) in enumerate(zip(self.params, self.exp_avg, self.exp_avg_sq)):
            g = p.grad
            if g is None or i in skip or (subset is not None and i not in subset):
                continue
            if not g.is_contiguous():
                g = g.contiguous()
            self.steps[i] += 1
            check(lib().ps_adam_step(_p(p), _p(g), _p(m), _p(v), p.numel(), self.lr, self.betas[0], self.betas[1], self.eps,
                                     self.weight_decay, self.steps[i], self.grad_scale, s), "ps_adam_step")

    def zero_grad(self):
        for p in self.params:
            if p.grad is not None:
                p.grad.zero_()

    def param_steps(self) -> List[int]:
        """torch's state[p]["step"] per parameter; the counts of device-decided groups (FlatGrads.define_groups) are read back
        from the device (one synchronising copy: checkpointing / tests only)"""
        out = list(self.steps)
        fg = getattr(self, "flat_grads", None)
        if fg is not None and fg.n_groups:
            dev = fg.group_steps.tolist()
            for i, p in enumerate(self.params):
                gr = getattr(p, "_ps_group", None)
                if gr is not None:
                    out[i] = dev[gr]
        return out

    def state_dict(self):
        """Checkpoint payload.  With a sharded gradient exchange every rank's moments are valid on its OWNED shard only: they
        are all-gathered here (a collective: call it on every rank), so that any rank's state_dict is complete."""
        fg = getattr(self, "flat_grads", None)
        if fg is not None and self.flat is not None:
            fg.gather_flat(self.flat[2])
            fg.gather_flat(self.flat[3])
        return {"step": self.step_count, "steps": self.param_steps(), "exp_avg": self.exp_avg, "exp_avg_sq": self.exp_avg_sq, "lr": self.lr}

    def load_state_dict(self, sd):
        self.step_count = sd["step"]
        self.steps = list(sd.get("steps", [sd["step"]] * len(self.params)))
        fg = getattr(self, "flat_grads", None)
        if fg is not None and fg.n_groups:
            host = fg.group_steps.tolist()
            for i, p in enumerate(self.params):
                gr = getattr(p, "_ps_group", None)
                if gr is not None:
                    host[gr] = self.steps[i]
            fg.group_steps.copy_(torch.tensor(host, dtype=torch.int32))
        for a, b in zip(self.exp_avg, sd["exp_avg"]):
            a.copy_(b)
        for a, b in zip(self.exp_avg_sq, sd["exp_avg_sq"]):
            a.copy_(b)


class WarmupMultiStepSchedule:
    """Learning-rate schedule of the PreSight method configs (ns/engine/my_schedulers.py:50-70 with the arguments of
    ns/configs/method_configs.py:158-168): torch's ChainedScheduler([LinearLR(start_factor=0.01, total_iters=warmup_steps),
    MultiStepLR(milestones, gamma=0.33)]) in closed form,
        lr(t) = lr_init * (0.01 + 0.99 * min(t, warmup) / warmup) * gamma ** #{m in milestones : m <= t},
    applied to a HipAdam by step(): call once after every optimizer step, like Optimizers.scheduler_step_all."""

    def __init__(self, optimizer: HipAdam, lr_init: Optional[float] = None, max_steps: int = 1000000,
                 milestones: Sequence[int] = (500000, 750000, 900000), warmup_steps: Optional[int] = None, gamma: float = 0.33,
                 start_factor: float = 0.01):
        self.opt = optimizer
        self.lr_init = optimizer.lr if lr_init is None else lr_init
        self.milestones = sorted(int(m) for m in milestones)
        self.warmup = int(warmup_steps) if warmup_steps else 0
        self.gamma, self.start_factor, self.max_steps = gamma, start_factor, max_steps
        self.t = 0
        self.opt.lr = self.lr_at(0)

    def lr_at(self, t: int) -> float:
        warm = 1.0 if self.warmup <= 0 else self.start_factor + (1.0 - self.start_factor) * min(t, self.warmup) / self.warmup
        return self.lr_init * warm * self.gamma ** sum(1 for m in self.milestones if m <= t)

    def step(self, step: Optional[int] = None) -> float:
        self.t = self.t + 1 if step is None else step + 1
        self.opt.lr = self.lr_at(self.t)
        return self.opt.lr

    def get_last_lr(self) -> List[float]:
        return [self.opt.lr]

    def state_dict(self):
        return {"t": self.t, "lr_init": self.lr_init}

    def load_state_dict(self, sd):
        self.t = int(sd["t"])
        self.lr_init = float(sd.get("lr_init", self.lr_init))
        self.opt.lr = self.lr_at(self.t)


# ------------------------------------------------------------------------------------------------ the orthogonalised update
NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)  # pushes (0, 1] into about [0.7, 1.2] in five steps: steep at zero, flat around one
NS_MAX_SIDE = 16384  # of the short side
_NS_MAX_TILES = (1 << 24) - 8  # of 64 x 64 over a whole stack: their launch holds fewer than 2^32 threads
_NS_BOUND = 15.0  # on squared singular values and on the polynomial: what the kernels' fp16 planes can hold (csrc/orthogonal.hip)


@functools.lru_cache(maxsize=64)
def _ns_check(steps: int, a: float, b: float, c: float) -> float:
    """the singular values of every iterate's S and of a + b S + c S^2, bounded from those of the first iterate (at most 1) -> the power
    of two that the latter stay under"""
    if not all(math.isfinite(v) for v in (a, b, c)):
        raise ValueError(f"presight_amd: the coefficients must be finite (got {(a, b, c)})")
    u, grow = 1.0, 1.0
    for _ in range(steps):
        t = u * u
        inner = [0.0, t] + ([-b / (2 * c)] if c != 0 and 0 < -b / (2 * c) < t else [])
        p = max(abs(a + b * v + c * v * v) for v in inner)
        # extremes of v (a + b v^2 + c v^4) on [0, u]: the ends and the roots of a + 3 b w + 5 c w^2, w = v^2
        roots: List[float] = []
        d = 9 * b * b - 20 * a * c
        if d >= 0:  # (as 2 a / h and h / (10 c), of which neither cancels; a very small c has one root far outside)
            h = -3 * b - math.copysign(math.sqrt(d), b)
            roots = [num / den for num, den in ((2 * a, h), (h, 10 * c)) if abs(num) < t * abs(den)]
        ends = [u] + [math.sqrt(w) for w in roots if 0 < w < t]
        u = max(abs(v * (a + b * v * v + c * v ** 4)) for v in ends)
        if max(p, u * u) > _NS_BOUND:
            raise ValueError(f"presight_amd: with coefficients {(a, b, c)} the iterates grow too large within {steps} steps")
        while grow < p:
            grow *= 2.0
    return grow


def _ns_args(steps: int, coefficients: Tuple[float, float, float], eps: float) -> Tuple[int, float, float, float, float, float]:
    if int(steps) != steps or not 1 <= steps <= 64:
        raise ValueError(f"presight_amd: 1 to 64 steps (got {steps})")
    if len(coefficients) != 3:
        raise ValueError(f"presight_amd: three coefficients (got {coefficients})")
    if not (math.isfinite(eps) and eps >= 0):
        raise ValueError(f"presight_amd: eps must be finite and not negative (got {eps})")
    a, b, c = (float(v) for v in coefficients)
    return int(steps), a, b, c, _ns_check(int(steps), a, b, c), float(eps)


def _matrices(t: torch.Tensor, name: str) -> Tuple[int, int, int]:
    if t.dim() < 2:
        raise ValueError(f"presight_amd: {name} must be a matrix or a stack of matrices (got shape {tuple(t.shape)})")
    m, n = t.shape[-2:]
    B = math.prod(t.shape[:-2])
    if min(m, n) > NS_MAX_SIDE or max(m, n) > 1 << 20 or B > 65535:
        raise ValueError(f"presight_amd: {name}: up to 65535 matrices of {NS_MAX_SIDE} x {1 << 20} (got shape {tuple(t.shape)})")
    if B * -(-m // 64) * -(-n // 64) >= _NS_MAX_TILES:
        raise ValueError(f"presight_amd: {name}: up to {_NS_MAX_TILES - 1} tiles of 64 x 64 in a stack (got shape {tuple(t.shape)})")
    return B, m, n


@torch.no_grad()
def newton_schulz(g: torch.Tensor, steps: int = 5, coefficients: Tuple[float, float, float] = NS_COEFFICIENTS, eps: float = 1e-7) -> torch.Tensor:
    """g [..., m, n] in fp32, fp16 or bf16 -> a tensor of its shape and type: every matrix scaled to X = G / (||G||_F + eps) and taken
    `steps` times through X <- a X + (b S + c S S) X with S = X X^T: its singular vectors kept, its singular values moved towards one.
    A matrix with a short side up to 64 is computed in fp32 where a workgroup's memory holds it (and it is not long, one of few); others as
    fp16 pairs: 22 bits of every entry, and what lies below 2^-27 of the matrix' norm to 2^-49 of it.  Sums in fp32, one rounding at the
    end.  The way and the tiles that a matrix takes go by its shape and by how many the stack holds: the same matrix may differ in its last bits
    between stacks of different length.  A zero matrix stays zero; a matrix with an infinite or
    undefined entry becomes undefined, without touching the others of the stack.  Not differentiable."""
    args = _ns_args(steps, tuple(coefficients), eps)
    code = _typed(_gpu(g, "g"), "g")
    B, m, n = _matrices(g, "g")
    g = g.contiguous()
    with _on(g.device):
        out = torch.empty_like(g)
        if out.numel():
            nbytes = lib().ps_newton_schulz_workspace(B, m, n)
            ws = torch.empty(nbytes, device=g.device, dtype=torch.uint8) if nbytes else None
            check(lib().ps_newton_schulz(_p(g), B, m, n, code, *args, _p(out), _p(ws), _stream()), "ps_newton_schulz")
    return out


def _with_gradients(params: Sequence[torch.nn.Parameter]) -> List[int]:
    """indices of the parameters that have received a gradient: of those whose gradient a FlatGrads holds, the ones it counts, which is the
    same on every rank.  Gradients written in place may still be on their way on a side stream, which autograd does not see: the
    current stream waits for it first.  A sharded exchange leaves no rank with a whole matrix's averaged gradient: refused."""
    held = [i for i, p in enumerate(params) if p.grad is not None]
    direct = [i for i in held if getattr(params[i], "_ps_direct_grad", False)]
    buffers = {i: flat_grads_of(params[i]) for i in direct}
    owners = list(dict.fromkeys(fg for fg in buffers.values() if fg is not None))  # (in the parameters' order: touched() may be a collective)
    for fg in owners:
        if fg.mode == "sharded" and fg._distributed() and fg._rank_world()[1] > 1:
            raise RuntimeError("HipMuon: in the sharded exchange a rank holds the averaged gradient of its shard only, and this update needs "
                               "whole matrices: exchange with mode='allreduce'")
    if direct:
        join_side_streams()
    counted = {id(p) for fg in owners for p, touched in zip(fg.params, fg.touched()) if touched}

    def received(i: int) -> bool:
        if i not in buffers:
            return True
        return params[i]._ps_touched if buffers[i] is None else id(params[i]) in counted

    return [i for i in held if received(i)]


class HipMuon:
    """Momentum with an orthogonalised update, for weight matrices [out, in] and stacks of them [experts, out, in] (embeddings, hash
    tables, biases and output scalars belong to HipAdam):
        buf <- momentum * buf + (1 - momentum) * grad
        u    = momentum * buf + (1 - momentum) * grad   (nesterov)   |   buf
        p   <- (1 - lr * weight_decay) * p - lr * scale * newton_schulz(u)
    scale: "spectral": sqrt(max(1, out / in)), an update whose effect on activations does not depend on the width;
           "rms": 0.2 * sqrt(max(out, in)), an update of the size Adam's has (its learning rates carry over).
    Parameters are contiguous fp32; one without a gradient is skipped, its momentum included.  lr may be changed between steps; a captured
    step keeps the lr, weight_decay and set of parameters it was captured with.
    Gradients held by a FlatGrads are read where it keeps them (a parameter counts as without a gradient from its zero_() until the backward
    pass has reached it; a step that is captured is captured together with that pass, whose side streams it waits for); parameters of its device-decided groups and gradients of its sharded exchange (a rank has its shard of a matrix only) are
    refused."""

    def __init__(self, params: Iterable[torch.nn.Parameter], lr: float = 0.02, momentum: float = 0.95, nesterov: bool = True,
                 weight_decay: float = 0.0, ns_steps: int = 5, ns_coefficients: Tuple[float, float, float] = NS_COEFFICIENTS, eps: float = 1e-7,
                 scale: str = "spectral"):
        self.params: List[torch.nn.Parameter] = [p for p in params if p.requires_grad and p.numel() > 0]
        for p in self.params:
            if not p.is_cuda or p.dtype != torch.float32 or not p.is_contiguous():
                raise RuntimeError("HipMuon: parameters must be contiguous fp32 CUDA tensors")
            _matrices(p, "a parameter")
        if len({id(p) for p in self.params}) != len(self.params):
            raise ValueError("HipMuon: a parameter appears more than once")
        if not 0.0 <= momentum < 1.0:
            raise ValueError(f"HipMuon: 0 <= momentum < 1 (got {momentum})")
        if scale not in ("spectral", "rms"):
            raise ValueError(f"HipMuon: scale is 'spectral' or 'rms' (got {scale!r})")
        self.lr, self.momentum, self.nesterov, self.weight_decay, self.scale = lr, momentum, nesterov, weight_decay, scale
        self.ns = _ns_args(ns_steps, tuple(ns_coefficients), eps)
        self.step_count = 0
        self.momentum_buffers = [torch.zeros_like(p, requires_grad=False) for p in self.params]

    def _rate(self, p: torch.Tensor) -> float:
        out, n_in = p.shape[-2:]
        return self.lr * (math.sqrt(max(1.0, out / n_in)) if self.scale == "spectral" else 0.2 * math.sqrt(max(out, n_in)))

    @torch.no_grad()
    def step(self) -> None:
        by_device: dict = {}
        for i in _with_gradients(self.params):
            p, buf = self.params[i], self.momentum_buffers[i]
            g = p.grad
            if getattr(p, "_ps_group", None) is not None:
                raise RuntimeError("HipMuon: whether this parameter has a gradient is decided on the device; it belongs to HipAdam")
            if p.device != buf.device or not p.is_contiguous() or p.dtype != torch.float32 or p.shape != buf.shape:
                raise RuntimeError("HipMuon: a parameter has changed its device, type, shape or layout since the optimizer was made")
            if g.layout != torch.strided or g.dtype != torch.float32 or g.device != p.device or g.shape != p.shape:
                raise RuntimeError("HipMuon: gradients must be dense fp32 tensors on their parameter's device")
            by_device.setdefault(p.device, []).append((p, g.contiguous(), buf))
        self.step_count += 1  # (a refused step is none)
        for device, stacks in by_device.items():
            k = len(stacks)
            sizes = [_matrices(p, "a parameter") for p, _, _ in stacks]
            i64, ptr = ctypes.c_int64 * k, ctypes.c_void_p * k
            with _on(device):
                nbytes = max(lib().ps_newton_schulz_workspace(*s) for s in sizes)
                ws = torch.empty(nbytes, device=device, dtype=torch.uint8) if nbytes else None
                check(lib().ps_muon_step(k, ptr(*[_p(s[0]) for s in stacks]), ptr(*[_p(s[1]) for s in stacks]), ptr(*[_p(s[2]) for s in stacks]),
                                         i64(*[s[0] for s in sizes]), i64(*[s[1] for s in sizes]), i64(*[s[2] for s in sizes]),
                                         (ctypes.c_float * k)(*[self._rate(s[0]) for s in stacks]), self.momentum, int(self.nesterov),
                                         1.0 - self.lr * self.weight_decay, *self.ns, _p(ws), _stream()), "ps_muon_step")

    def zero_grad(self):
        for p in self.params:
            if p.grad is not None:
                p.grad.zero_()

    def state_dict(self):
        return {"step": self.step_count, "lr": self.lr, "momentum_buffers": self.momentum_buffers}

    def load_state_dict(self, sd):
        here, there = ([tuple(b.shape) for b in bufs] for bufs in (self.momentum_buffers, sd["momentum_buffers"]))
        if here != there:  # (copy_ would spread a smaller one over a stack)
            raise ValueError(f"HipMuon: the state is of other parameters: shapes {there} for {here}")
        self.step_count, self.lr = sd["step"], sd["lr"]
        for a, b in zip(self.momentum_buffers, sd["momentum_buffers"]):
            a.copy_(b)
