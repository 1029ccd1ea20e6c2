"""Routing of tokens to experts and the sum of what the experts return.  Not in the reference: with expert_linear these
are the layer between two attention cores of a mixture-of-experts model.

    weights, experts = route(logits, top_k)               T x top_k each
    plan = dispatch(experts, num_experts)                 the tokens' slots sorted by expert
    y = expert_linear(x, codes, scales, fmt, plan)        a row a slot, in the experts' order
    out = combine(y, weights, plan, residual=shared)      T x D

route and combine are differentiable once and in reverse mode, in the logits, and in y, the weights and the residual.
"""
from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from .. import _lib

__all__ = ["route", "dispatch", "combine", "Dispatch", "SCORES"]

SCORES = ("softmax", "sigmoid")
MAX_EXPERTS, MAX_TOP_K, MAX_GROUPS = 1024, 64, 64
_DTYPES = _lib.DTYPE_CODE


def _dtype(t: torch.Tensor, who: str, what: str) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"mxq.nn.{who}: {what} must be float32, bfloat16 or float16, got {t.dtype}")
    return code


def _no_tangent(who: str, *tensors: Optional[torch.Tensor]) -> None:
    """Refuses inputs of forward-mode differentiation, which do not ask for a gradient and whose tangent a kernel on
    raw pointers would drop."""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"mxq.nn.{who}: no forward-mode derivative")


def _whole(value, who: str, what: str, low: int, high: int) -> int:
    if isinstance(value, bool) or not isinstance(value, int) or not low <= value <= high:
        raise ValueError(f"mxq.nn.{who}: {what} must be an integer from {low} to {high}, got {value!r}")
    return value


def _once(backward):
    """once_differentiable, without its context where no graph of the gradient is asked for."""
    guarded = once_differentiable(backward)

    def run(ctx, *grads):
        return (guarded if torch.is_grad_enabled() else backward)(ctx, *grads)
    return run


@_lib.memo_spec
def _route_spec(E, top_k, score, groups, top_groups, renormalize, scale):
    _whole(E, "route", "the number of experts", 1, MAX_EXPERTS)
    _whole(top_k, "route", "top_k", 1, min(MAX_TOP_K, E))
    _whole(groups, "route", "groups", 1, min(MAX_GROUPS, E))
    if E % groups:
        raise ValueError(f"mxq.nn.route: groups {groups} must divide the {E} experts")
    _whole(top_groups, "route", "top_groups", 1, groups)
    if score not in SCORES:
        raise ValueError(f"mxq.nn.route: score must be one of {SCORES}, got {score!r}")
    return _lib.RouteSpec(SCORES.index(score), top_k, groups, top_groups, int(bool(renormalize)), float(scale))


def _route(logits, bias, spec):
    T, E = logits.shape
    dev = logits.device
    weights = logits.new_empty((T, spec.top_k), dtype=torch.float32)
    experts = logits.new_empty((T, spec.top_k), dtype=torch.int32)
    with _lib.on(dev):
        _lib.run("mxq_route", logits.data_ptr(), _DTYPES[logits.dtype], _lib.ptr(bias), T, E, spec, weights.data_ptr(),
                 experts.data_ptr(), _lib.stream(dev))
    return weights, experts


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, spec):
        weights, experts = _route(logits, bias, spec)
        ctx.save_for_backward(logits, experts)
        ctx.spec = spec
        ctx.mark_non_differentiable(experts)
        ctx.set_materialize_grads(False)               # the experts' would be a tensor of zeros
        return weights, experts

    @staticmethod
    @_once
    def backward(ctx, grad, _):
        if grad is None:
            return None, None, None
        logits, experts = ctx.saved_tensors
        dev = logits.device
        grad = grad.to(torch.float32).contiguous()
        out = torch.empty_like(logits)
        with _lib.on(dev):
            _lib.run("mxq_route_grad", logits.data_ptr(), _DTYPES[logits.dtype], experts.data_ptr(), grad.data_ptr(),
                     logits.shape[0], logits.shape[1], ctx.spec, out.data_ptr(), _lib.stream(dev))
        return out, None, None


def route(logits: torch.Tensor, top_k: int, *, score: str = "softmax", bias: Optional[torch.Tensor] = None,
          groups: int = 1, top_groups: int = 1, renormalize: bool = True,
          scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(weights float32, experts int32), ... x top_k each, of logits ... x E, best first, ties to the lowest index.

    score: "softmax" over the experts or "sigmoid" of each.  bias (E values): added to the scores for the choice, not
    to the weights; no gradient.  groups: E / groups neighbouring experts form a group, and only the top_groups groups
    with the largest sum of their two best (biased) scores are open.  renormalize: the chosen scores are divided by
    their sum.  scale multiplies the weights.

    A logit of -inf closes its expert.  Where fewer than top_k are open the rest is expert -1 with weight 0, which
    dispatch leaves out.  A row with a NaN (for softmax also +inf) gets NaN weights and experts -1, and a gradient of
    NaN; a NaN of the bias does the same to the weights, and leaves no gradient, as all slots of no expert.  Scores are taken
    in 64 bits, so that the choice does not depend on float32's rounding of exp."""
    _dtype(logits, "route", "logits")
    if logits.ndim < 1:
        raise ValueError("mxq.nn.route: logits must have an experts axis")
    E = logits.shape[-1]
    spec = _route_spec(E, top_k, score, groups, top_groups, renormalize, scale)
    _no_tangent("route", logits)
    if bias is not None and tuple(bias.shape) != (E,):
        raise ValueError(f"mxq.nn.route: bias must hold {E} values, got shape {tuple(bias.shape)}")
    dev = _lib.compute_device(logits)
    if bias is not None:
        bias = _lib.to_device(bias.detach(), dev).to(torch.float32).contiguous()
    flat = logits if logits.ndim == 2 else logits.reshape(-1, E)
    flat = _lib.to_device(flat, dev).contiguous()
    grad = flat.requires_grad and torch.is_grad_enabled()
    weights, experts = (_Route.apply if grad else _route)(flat, bias, spec)
    if logits.ndim != 2:
        lead = logits.shape[:-1]
        weights, experts = weights.reshape(*lead, top_k), experts.reshape(*lead, top_k)
    return _lib.back(weights, logits), _lib.back(experts, logits)


class Dispatch(NamedTuple):
    """The slots (slot t * top_k + j: token t's j-th choice) in the experts' order.  order (n): the slot of each row;
    offsets (num_experts + 1): each expert's first row; positions (tokens x top_k): the row of each slot, -1 - row for
    a slot of no expert, whose rows come last.  All int32, on the experts' device."""
    order: torch.Tensor
    offsets: torch.Tensor
    positions: torch.Tensor

    @property
    def num_experts(self) -> int:
        return self.offsets.shape[0] - 1

    @property
    def top_k(self) -> int:
        return self.positions.shape[1]


def dispatch(experts: torch.Tensor, num_experts: int) -> Dispatch:
    """Sorts the slots of experts (tokens x top_k whole numbers) by expert, equal ones in the order of their tokens.
    A slot whose expert is not in [0, num_experts) belongs to none."""
    if experts.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"mxq.nn.dispatch: experts must be int32 or int64, got {experts.dtype}")
    if experts.ndim != 2 or not 1 <= experts.shape[1] <= MAX_TOP_K:
        raise ValueError(f"mxq.nn.dispatch: experts must be tokens x top_k, top_k from 1 to {MAX_TOP_K}, got shape "
                         f"{tuple(experts.shape)}")
    _whole(num_experts, "dispatch", "num_experts", 1, MAX_EXPERTS)
    dev = _lib.compute_device(experts)
    e = _lib.to_device(experts.detach(), dev)
    if e.dtype == torch.int64:
        e = e.clamp(-1, num_experts).to(torch.int32)             # a far index must not wrap into the range
    e = e.contiguous()
    n = e.numel()
    order = e.new_empty(n, dtype=torch.int32)
    offsets = e.new_empty(num_experts + 1, dtype=torch.int32)
    positions = torch.empty_like(e)
    with _lib.on(dev):
        _lib.run("mxq_dispatch", e.data_ptr(), n, num_experts, order.data_ptr(), offsets.data_ptr(),
                 positions.data_ptr(), _lib.stream(dev))
    return Dispatch(_lib.back(order, experts), _lib.back(offsets, experts), _lib.back(positions, experts))


def _check_plan(plan, who: str) -> None:
    if not isinstance(plan, Dispatch):
        raise TypeError(f"mxq.nn.{who}: plan must be dispatch's, got {type(plan).__name__}")
    order, offsets, positions = plan
    if order.dtype != torch.int32 or offsets.dtype != torch.int32 or positions.dtype != torch.int32 or \
            positions.ndim != 2 or order.ndim != 1 or len(order) != positions.numel() or offsets.ndim != 1 or \
            len(offsets) < 2:
        raise ValueError(f"mxq.nn.{who}: plan does not hold dispatch's tensors")


def _combine(y, weights, positions, residual):
    T, k = positions.shape
    D, dev = y.shape[1], y.device
    out = y.new_empty((T, D))
    with _lib.on(dev):
        _lib.run("mxq_combine", y.data_ptr(), _DTYPES[y.dtype], weights.data_ptr(), positions.data_ptr(),
                 _lib.ptr(residual), out.data_ptr(), T, k, D, _lib.stream(dev))
    return out


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, positions, residual):
        out = _combine(y, weights, positions, residual)
        ctx.save_for_backward(y, weights, positions)
        return out

    @staticmethod
    @_once
    def backward(ctx, grad):
        y, weights, positions = ctx.saved_tensors
        T, k = positions.shape
        dev = y.device
        grad = grad.contiguous()
        dy = torch.empty_like(y) if ctx.needs_input_grad[0] else None
        dw = torch.empty_like(weights) if ctx.needs_input_grad[1] else None
        with _lib.on(dev):
            _lib.run("mxq_combine_grad", _lib.ptr(grad), _DTYPES[y.dtype], _lib.ptr(y), _lib.ptr(weights),
                     _lib.ptr(positions), _lib.ptr(dy), _lib.ptr(dw), T, k, y.shape[1], _lib.stream(dev))
        return dy, dw, None, grad if ctx.needs_input_grad[3] else None


def combine(y: torch.Tensor, weights: torch.Tensor, plan: Dispatch,
            residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """residual + sum_j weights[t, j] * (the row of y that token t's j-th slot has in plan): tokens x D in y's dtype.

    y: n x D in the experts' order.  The sum is float32, in the order of j, and rounded once.  A slot of no expert adds
    nothing, unless its weight is NaN, which the token's output then is; a position past y's rows, which no plan of
    dispatch's holds, is taken as one of no expert."""
    _check_plan(plan, "combine")
    _dtype(y, "combine", "y")
    T, k = plan.positions.shape
    if y.ndim != 2 or y.shape[0] != T * k:
        raise ValueError(f"mxq.nn.combine: y must have {T * k} rows, one a slot, got shape {tuple(y.shape)}")
    if tuple(weights.shape) != (T, k) or not weights.is_floating_point():
        raise ValueError(f"mxq.nn.combine: weights must be {T} x {k} floating, got {tuple(weights.shape)} "
                         f"{weights.dtype}")
    if residual is not None and (tuple(residual.shape) != (T, y.shape[1]) or residual.dtype != y.dtype):
        raise ValueError(f"mxq.nn.combine: residual must be {T} x {y.shape[1]} {y.dtype}, got "
                         f"{tuple(residual.shape)} {residual.dtype}")
    _no_tangent("combine", y, weights, residual)
    dev = _lib.compute_device(y, weights)
    yd = _lib.to_device(y, dev).contiguous()
    wd = _lib.to_device(weights, dev).to(torch.float32).contiguous()
    pd = _lib.to_device(plan.positions, dev).contiguous()
    rd = None if residual is None else _lib.to_device(residual, dev).contiguous()
    grad = torch.is_grad_enabled() and (yd.requires_grad or wd.requires_grad or (rd is not None and rd.requires_grad))
    return _lib.back((_Combine.apply if grad else _combine)(yd, wd, pd, rd), y)
