"""Rows sorted by expert and back, and the experts' linear layers on the sorted rows (a mixture of experts: the soft form of the routed
sub-fields, which send every point to its nearest sub-field alone).

    plan = expert_plan(ids, E)                       # ids [N, k]: the experts of every row; outside [0, E): no expert
    rows = expert_dispatch(x, plan)                  # x [N, D] -> [N*k, D], sorted by expert
    h    = expert_linear(rows, weight, bias, plan)   # weight [E, out, in]: h[p] = W_e rows[p] + b_e
    y    = expert_combine(h, gates, plan)            # gates [N, k] -> [N, out]: y[n] = sum_j gates[n, j] h[place of (n, j)]

Everything is asynchronous on the current stream of the tensors' device, nothing synchronises with the host, and all results are
independent of timing (no atomics on values): calls can be captured into a graph.  Differentiable once with respect to x, weight, bias,
rows and gates.  Element types fp32, fp16 and bf16; every sum is held in fp32 and rounded once.  Rows of the sorted layout behind the
last expert's (one for every assignment to no expert) are zero in every result and are never read.

Capturing a backward pass: an eager graph of the same leaves that is still alive keeps its gradient accumulation nodes on the stream
they were made on, and a capture that reaches them fails.  Capture torch.autograd.grad (which has no such nodes), or drop the eager graph
before the capture."""
from __future__ import annotations

import contextlib
from typing import Optional, Union

import torch
from torch import Tensor
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from ._lib import check, lib
from .ops import _p, _stream

DTYPE_CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
MAX_EXPERTS = 1024
MAX_WIDTH = 1 << 20


def _on(device: torch.device):
    """launches go to `device`, whatever device is current"""
    return contextlib.nullcontext() if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _gpu(t: Tensor, name: str, device: Optional[torch.device] = None) -> Tensor:
    if not isinstance(t, Tensor):
        raise TypeError(f"presight_amd: {name} must be a tensor (got {type(t).__name__})")
    if not t.is_cuda:
        raise RuntimeError(f"presight_amd: {name} must live on the GPU (got {t.device}); the HIP path has no CPU fallback")
    if device is not None and t.device != device:
        raise RuntimeError(f"presight_amd: {name} is on {t.device}, the other tensors are on {device}")
    return t


def _typed(t: Tensor, name: str) -> int:
    if t.dtype not in DTYPE_CODES:
        raise TypeError(f"presight_amd: {name} must be float32, float16 or bfloat16 (got {t.dtype})")
    return DTYPE_CODES[t.dtype]


def _rows(t: Tensor) -> Tensor:
    """rows of consecutive elements, at any distance from each other; other layouts are copied"""
    return t if t.shape[1] <= 1 or t.stride(1) == 1 else t.contiguous()


def _wants_grad(*tensors) -> bool:
    """whether a call goes through autograd: to be differentiated, or to be refused by it where an input carries a forward-mode tangent"""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        return True
    return forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _once(fn):
    """differentiable once: torch's guard, where second derivatives are being recorded (it costs as much as a small kernel otherwise)"""
    guarded = once_differentiable(fn)
    return lambda ctx, *grads: (guarded if torch.is_grad_enabled() else fn)(ctx, *grads)


class ExpertPlan:
    """Who goes where, for ids [N, k] and E experts (contiguous int32 tensors on the ids' device):
        offsets [E+1]   expert e's rows are the sorted places offsets[e] .. offsets[e+1]
        src     [N*k]   sorted place -> assignment n*k + j, in order of (expert, assignment); -1 behind offsets[E]
        dst     [N, k]  assignment -> sorted place; -1: to no expert
    One made by hand has to hold what expert_plan would: every place once.  (Places outside [0, N*k) count as no expert.)"""

    def __init__(self, offsets: Tensor, src: Tensor, dst: Tensor, num_experts: int):
        if dst.dim() != 2 or offsets.shape != (num_experts + 1,) or src.shape != (dst.numel(),):
            raise ValueError(f"presight_amd: a plan for {num_experts} experts holds offsets [{num_experts + 1}], src [rows * k] and dst [rows, k] "
                             f"(got {tuple(offsets.shape)}, {tuple(src.shape)}, {tuple(dst.shape)})")
        for t in (offsets, src, dst):
            if t.dtype != torch.int32 or t.device != dst.device or not t.is_contiguous():
                raise TypeError("presight_amd: a plan holds contiguous int32 tensors on one device")
        self._set(offsets, src, dst, num_experts)

    def _set(self, offsets: Tensor, src: Tensor, dst: Tensor, num_experts: int) -> "ExpertPlan":
        self.offsets, self.src, self.dst, self.num_experts = offsets, src, dst, num_experts
        self.num_rows, self.k = dst.shape
        return self

    @property
    def num_places(self) -> int:
        return self.num_rows * self.k

    @property
    def held(self) -> Tensor:
        """number of assignments to an expert (a device scalar, no synchronisation)"""
        return self.offsets[self.num_experts:]


def expert_plan(ids: Tensor, num_experts: int) -> ExpertPlan:
    """ids [N, k] int32 or int64.  An expert may be named twice by one row: those are two assignments."""
    _gpu(ids, "ids")
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"presight_amd: ids must be int32 or int64 (got {ids.dtype})")
    if ids.dim() != 2 or ids.shape[1] < 1:
        raise ValueError(f"presight_amd: ids must be [rows, k] with k >= 1 (got {tuple(ids.shape)})")
    if not 1 <= num_experts <= MAX_EXPERTS:
        raise ValueError(f"presight_amd: 1 to {MAX_EXPERTS} experts (got {num_experts})")
    ids = ids.contiguous()
    N, k = ids.shape
    M, dev = N * k, ids.device
    if M >= 2 ** 31 - 2 ** 20:
        raise ValueError(f"presight_amd: {M} assignments do not fit 32-bit places")
    with _on(dev):
        offsets = torch.empty(num_experts + 1, device=dev, dtype=torch.int32)
        src = torch.empty(M, device=dev, dtype=torch.int32)
        dst = torch.empty(N, k, device=dev, dtype=torch.int32)
        ints = lib().ps_expert_plan_workspace(M, num_experts)
        ws = torch.empty(ints, device=dev, dtype=torch.int32) if ints else None
        check(lib().ps_expert_plan(_p(ids), int(ids.dtype == torch.int64), M, num_experts, _p(offsets), _p(src), _p(dst), _p(ws), _stream()),
              "ps_expert_plan")
    return ExpertPlan.__new__(ExpertPlan)._set(offsets, src, dst, num_experts)


# ------------------------------------------------------------------------------------------------ exchange
def _dispatch(x: Tensor, dst: Tensor, offsets: Tensor) -> Tensor:
    x = _rows(x)
    (N, k), D = dst.shape, x.shape[1]
    with _on(x.device):
        rows = torch.empty(N * k, D, device=x.device, dtype=x.dtype)
        check(lib().ps_expert_dispatch(_p(x), x.stride(0), _p(dst), _held(offsets), N, k, D, DTYPE_CODES[x.dtype], _p(rows), _stream()),
              "ps_expert_dispatch")
    return rows


def _combine(rows: Tensor, weights: Optional[Tensor], dst: Tensor) -> Tensor:
    rows = _rows(rows)
    (N, k), D = dst.shape, rows.shape[1]
    with _on(rows.device):
        y = torch.empty(N, D, device=rows.device, dtype=rows.dtype)
        check(lib().ps_expert_combine(_p(rows), rows.stride(0), _p(weights), _p(dst), N, k, D, DTYPE_CODES[rows.dtype], _p(y), _stream()),
              "ps_expert_combine")
    return y


def _held(offsets: Tensor) -> int:
    """address of the number of assignments to an expert"""
    return offsets.data_ptr() + 4 * (offsets.shape[0] - 1)


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dst, offsets):
        ctx.save_for_backward(dst)
        return _dispatch(x, dst, offsets)

    @staticmethod
    @_once
    def backward(ctx, drows):
        (dst,) = ctx.saved_tensors
        return _combine(drows, None, dst), None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, dst, offsets):
        w = None if weights is None else weights.detach().float().contiguous()
        ctx.save_for_backward(rows, w, dst, offsets)
        ctx.weights_dtype = None if weights is None else weights.dtype
        return _combine(rows, w, dst)

    @staticmethod
    @_once
    def backward(ctx, dy):
        rows, w, dst, offsets = ctx.saved_tensors
        if w is None:
            return _dispatch(dy, dst, offsets), None, None, None
        dy, rows = _rows(dy), _rows(rows)
        (N, k), D = dst.shape, rows.shape[1]
        with _on(rows.device):
            drows = torch.empty(rows.shape, device=rows.device, dtype=rows.dtype) if ctx.needs_input_grad[0] else None
            dw = torch.empty(N, k, device=rows.device, dtype=torch.float32) if ctx.needs_input_grad[1] else None
            check(lib().ps_expert_combine_bwd(_p(dy), dy.stride(0), _p(rows), rows.stride(0), _p(w), _p(dst), _held(offsets), N, k, D,
                                              DTYPE_CODES[rows.dtype], _p(drows), _p(dw), _stream()), "ps_expert_combine_bwd")
        return drows, None if dw is None else dw.to(ctx.weights_dtype), None, None


def _check_plan(plan) -> ExpertPlan:
    if not isinstance(plan, ExpertPlan):
        raise TypeError(f"presight_amd: plan must be an ExpertPlan (got {type(plan).__name__})")
    return plan


def expert_dispatch(x: Tensor, plan: ExpertPlan) -> Tensor:
    """x [N, D] -> rows [N*k, D]: row p is x[src[p] // k], zeros behind offsets[E]."""
    _check_plan(plan)
    _typed(_gpu(x, "x", plan.dst.device), "x")
    if x.dim() != 2 or x.shape[0] != plan.num_rows:
        raise ValueError(f"presight_amd: x must be [{plan.num_rows}, features] for this plan (got {tuple(x.shape)})")
    return _Dispatch.apply(x, plan.dst, plan.offsets) if _wants_grad(x) else _dispatch(x, plan.dst, plan.offsets)


def expert_combine(rows: Tensor, weights: Optional[Tensor], plan: ExpertPlan) -> Tensor:
    """rows [N*k, D], weights [N, k] (None: all ones) -> y [N, D], y[n] = sum_j weights[n, j] * rows[dst[n, j]], without the assignments
    to no expert, whose weights are not read.  Summed in fp32; the weights' gradient comes in the weights' type."""
    _check_plan(plan)
    _typed(_gpu(rows, "rows", plan.dst.device), "rows")
    if rows.dim() != 2 or rows.shape[0] != plan.num_places:
        raise ValueError(f"presight_amd: rows must be [{plan.num_places}, features] for this plan (got {tuple(rows.shape)})")
    if weights is not None:
        _typed(_gpu(weights, "weights", plan.dst.device), "weights")
        if tuple(weights.shape) != (plan.num_rows, plan.k):
            raise ValueError(f"presight_amd: weights must be {(plan.num_rows, plan.k)} for this plan (got {tuple(weights.shape)})")
    if not _wants_grad(rows, weights):
        return _combine(rows, None if weights is None else weights.float().contiguous(), plan.dst)
    return _Combine.apply(rows, weights, plan.dst, plan.offsets)


# ------------------------------------------------------------------------------------------------ the experts' linear layers
def _spaced(t: Tensor) -> Tensor:
    """rows that neither overlap nor lie further apart than the products' tiles can address (an expanded gradient is copied)"""
    t = _rows(t)
    return t if t.shape[0] <= 1 or t.shape[1] <= t.stride(0) <= MAX_WIDTH else t.contiguous()


def _ld(t: Tensor) -> int:
    return max(t.stride(0), t.shape[1]) if t.shape[0] > 1 else t.shape[1]


def _workspace(pass_: int, a: Tensor, b: Tensor, b_ld: int, M: int, E: int, n_in: int, n_out: int, code: int) -> Optional[Tensor]:
    nbytes = lib().ps_expert_linear_workspace(pass_, a.data_ptr(), _ld(a), b.data_ptr(), b_ld, M, E, n_in, n_out, code)
    return torch.empty(nbytes, device=a.device, dtype=torch.uint8) if nbytes else None


def _linear_fwd(x: Tensor, weight: Tensor, bias: Optional[Tensor], offsets: Tensor) -> Tensor:
    (M, n_in), (E, n_out, _) = x.shape, weight.shape
    code = DTYPE_CODES[x.dtype]
    x, weight = _spaced(x), weight.contiguous()
    if bias is not None:
        bias = bias.contiguous()
    with _on(x.device):
        y = torch.empty(M, n_out, device=x.device, dtype=x.dtype)
        ws = _workspace(0, x, weight, n_in, M, E, n_in, n_out, code)
        check(lib().ps_expert_linear_fwd(_p(x), _ld(x), _p(weight), _p(bias), _p(offsets), M, E, n_in, n_out, code, _p(y), _p(ws), _stream()),
              "ps_expert_linear_fwd")
    return y


class _ExpertLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, offsets):
        ctx.save_for_backward(x, weight, offsets)
        return _linear_fwd(x, weight, bias, offsets)

    @staticmethod
    @_once
    def backward(ctx, dy):
        x, weight, offsets = ctx.saved_tensors
        (M, n_in), (E, n_out, _) = x.shape, weight.shape
        code = DTYPE_CODES[x.dtype]
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        dx = dw = db = None
        with _on(x.device):
            dy = _spaced(dy)
            if need_x:
                w = weight.contiguous()
                dx = torch.empty(M, n_in, device=x.device, dtype=x.dtype)
                ws = _workspace(1, dy, w, n_in, M, E, n_in, n_out, code)
                check(lib().ps_expert_linear_dx(_p(dy), _ld(dy), _p(w), _p(offsets), M, E, n_in, n_out, code, _p(dx), _p(ws), _stream()),
                      "ps_expert_linear_dx")
            if need_w or need_b:
                xs = _spaced(x)
                dw = torch.empty(E, n_out, n_in, device=x.device, dtype=x.dtype)
                db = torch.empty(E, n_out, device=x.device, dtype=x.dtype) if need_b else None
                ws = _workspace(2, dy, xs, _ld(xs), M, E, n_in, n_out, code)
                check(lib().ps_expert_linear_dw(_p(dy), _ld(dy), _p(xs), _ld(xs), _p(offsets), M, E, n_in, n_out, code, _p(dw), _p(db), _p(ws),
                                                _stream()), "ps_expert_linear_dw")
        return dx, dw if need_w else None, db, None


def _offsets32(offsets: Tensor, M: int) -> Tensor:
    """as the kernels read them: those of a longer list may lie beyond 32 bits, and mean "behind the M rows" there too"""
    return (offsets if offsets.dtype == torch.int32 else offsets.clamp(0, M).to(torch.int32)).contiguous()


def expert_linear(x: Tensor, weight: Tensor, bias: Optional[Tensor], offsets: Union[Tensor, ExpertPlan]) -> Tensor:
    """x [M, in] sorted by expert, weight [E, out, in], bias [E, out] or None -> y [M, out], y[p] = weight[e] x[p] + bias[e] for the rows
    p in offsets[e] .. offsets[e+1].  offsets: an ExpertPlan, or int32 / int64 [E+1], ascending (others give undefined rows, within the
    results); a piece of a longer plan's offsets takes the experts of that piece.  Rows that belong to none of them are zero in y and in x's gradient and do not enter the others;
    experts without rows have zero gradients."""
    plan = offsets
    offsets = plan.offsets if isinstance(plan, ExpertPlan) else plan
    _typed(_gpu(x, "x"), "x")
    _gpu(weight, "weight", x.device), _gpu(offsets, "offsets", x.device)
    if bias is not None:
        _gpu(bias, "bias", x.device)
    if weight.dtype != x.dtype or (bias is not None and bias.dtype != x.dtype):
        raise TypeError(f"presight_amd: expert_linear takes x, weight and bias of one type (got {x.dtype}, {weight.dtype}"
                        f"{'' if bias is None else f', {bias.dtype}'})")
    if x.dim() != 2 or weight.dim() != 3 or weight.shape[2] != x.shape[1] or min(weight.shape) < 1:
        raise ValueError(f"presight_amd: expert_linear takes x [rows, in] and weight [experts, out, in] (got {tuple(x.shape)}, {tuple(weight.shape)})")
    if bias is not None and tuple(bias.shape) != tuple(weight.shape[:2]):
        raise ValueError(f"presight_amd: bias must be {tuple(weight.shape[:2])} (got {tuple(bias.shape)})")
    if offsets.dtype not in (torch.int32, torch.int64) or offsets.dim() != 1 or offsets.shape[0] != weight.shape[0] + 1:
        raise ValueError(f"presight_amd: offsets must be int32 or int64 [{weight.shape[0] + 1}] (got {offsets.dtype} {tuple(offsets.shape)})")
    if isinstance(plan, ExpertPlan) and x.shape[0] != plan.num_places:
        raise ValueError(f"presight_amd: x must have the plan's {plan.num_places} rows (got {x.shape[0]})")
    if max(weight.shape[1:]) > MAX_WIDTH or weight.shape[0] > 65536:
        raise ValueError("presight_amd: expert_linear takes up to 65536 experts and 2**20 features")
    offsets = _offsets32(offsets, x.shape[0])
    if not _wants_grad(x, weight, bias):
        return _linear_fwd(x, weight, bias, offsets)
    return _ExpertLinear.apply(x, weight, bias, offsets)
