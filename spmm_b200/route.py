"""Expert choice and the way back: ``route_topk`` and ``route_combine``.

``route_topk`` chooses each token's experts from router logits, weighs them,
and groups the chosen rows by expert (a ``Routing``) for ``grouped_matmul``;
``route_combine`` sums the experts' results back in token order.  Everything
stays on the device: no call waits for the GPU.  Not in the reference.
"""

from __future__ import annotations

import ctypes as C
import struct
from dataclasses import dataclass
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib
from ._device import on_device, stream_handle

__all__ = ['Routing', 'route_topk', 'route_topk_backward', 'route_combine', 'route_combine_backward', 'SCORINGS']

SCORINGS = ('softmax', 'sigmoid')
_TYPES = {torch.float32: _lib.DENSE_F32, torch.bfloat16: _lib.DENSE_BF16, torch.float16: _lib.DENSE_F16}


@dataclass(frozen=True, eq=False)
class Routing:
    """Rows grouped by expert, all int32 on one CUDA device.

    ``experts`` [T, k]: each token's experts, best first (-1: none).
    ``slots`` [T, k]: the row of the grouped order that each choice got (-1: none).
    ``rows`` [T*k]: the token of each row of the grouped order, ascending within
    an expert; -1 behind the last expert's rows.
    ``offsets`` [E+1]: the first row of each expert, and the end of the last one.

    ``route_topk`` makes one; in one of your own no row may have two choices
    (two slots alike): the gradients give each row one choice's values.  A
    choice is dropped by a slot of -1: its row then adds nothing and gets no
    gradient from ``route_combine``.
    """

    experts: torch.Tensor
    slots: torch.Tensor
    rows: torch.Tensor
    offsets: torch.Tensor

    @property
    def tokens(self) -> int:
        return self.slots.shape[0]

    @property
    def top(self) -> int:
        return self.slots.shape[1]

    @property
    def num_experts(self) -> int:
        return self.offsets.shape[0] - 1


def check_routing(r, device=None) -> None:
    if not isinstance(r, Routing):
        raise TypeError(f'routing must be a Routing, got {type(r).__name__}')
    index = None if device is None else -1 if device.index is None else device.index
    for name, dim in (('experts', 2), ('slots', 2), ('rows', 1), ('offsets', 1)):
        t = getattr(r, name)
        if not isinstance(t, torch.Tensor) or t.dtype is not torch.int32 or t.dim() != dim or not t.is_contiguous():
            raise ValueError(f'routing.{name} must be a contiguous {dim}D int32 tensor')
        if index is not None and t.get_device() != index:
            raise ValueError('routing must be on the operands\' device')
    if r.experts.shape != r.slots.shape or r.rows.shape[0] != r.slots.numel() or r.offsets.shape[0] < 2:
        raise ValueError('routing arrays do not belong together')


def need_cuda(t: torch.Tensor, what: str) -> None:
    if not t.is_cuda:
        raise ValueError(f'{what} must be a dense CUDA tensor')


def refuse_tangents(**tensors: Optional[torch.Tensor]) -> None:
    """The operators are differentiable backwards only; without this a tangent would be lost silently.  Called where
    forward_ad._current_level says that there can be one."""
    for name, t in tensors.items():
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f'{name} has a tangent: there are no forward-mode derivatives')


def _check_score(logits, scoring):
    if scoring not in SCORINGS:
        raise ValueError(f'scoring must be one of {SCORINGS}')
    if logits.dim() != 2 or logits.layout != torch.strided:
        raise ValueError(f'logits must be a dense 2D tensor, got {logits.dim()}D')
    if logits.dtype not in _TYPES:
        raise TypeError(f'logits must be float32, bfloat16 or float16, got {logits.dtype}')


def _unit_rows(t: torch.Tensor) -> torch.Tensor:
    """`t` with unit stride along its last dimension."""
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


# spmm_route_args and spmm_combine_args (include/spmm_b200.h) packed in one go, see linear.py
_ROUTE = struct.Struct('@4i3qPqPfi8PQ').pack
_COMBINE = struct.Struct('@2i5q9P5q').pack
assert struct.calcsize('@4i3qPqPfi8PQ') == C.sizeof(_lib.RouteArgs)
assert struct.calcsize('@2i5q9P5q') == C.sizeof(_lib.CombineArgs)


def _topk(logits, top, scoring, renormalize, scale, bias):
    logits = _unit_rows(logits)
    device = logits.device
    tokens, experts = logits.shape
    L = _lib.lib()
    head = (1, _TYPES[logits.dtype], SCORINGS.index(scoring), int(bool(renormalize)), tokens, experts, top,
            logits.data_ptr(), logits.stride(0), 0 if bias is None else bias.data_ptr(), scale, 0)
    with on_device(device):
        weights = logits.new_empty((tokens, top), dtype=torch.float32)
        chosen = logits.new_empty((tokens, top), dtype=torch.int32)
        slots = torch.empty_like(chosen)
        rows = chosen.new_empty(tokens * top)
        offsets = chosen.new_empty(experts + 1)
        args = head + (weights.data_ptr(), chosen.data_ptr(), slots.data_ptr(), rows.data_ptr(), offsets.data_ptr(),
                       0, 0)
        stream = stream_handle(device)
        n = L.spmm_route_workspace_size(_ROUTE(*args, 0, 0))
        ws = chosen.new_empty(n // 4) if n else None
        rc = L.spmm_route(_ROUTE(*args, ws.data_ptr() if n else 0, n), stream)
        _lib.check(rc, 'route_topk')
    return weights, chosen, slots, rows, offsets


def _topk_backward(dweights, logits, experts, scoring, renormalize, scale):
    logits, dweights = _unit_rows(logits), dweights.contiguous()
    device = logits.device
    with on_device(device):
        out = logits.new_empty(logits.shape)
        args = _ROUTE(1, _TYPES[logits.dtype], SCORINGS.index(scoring), int(bool(renormalize)), *logits.shape,
                      experts.shape[1], logits.data_ptr(), logits.stride(0), 0, scale, 0, 0, experts.data_ptr(), 0, 0,
                      0, dweights.data_ptr(), out.data_ptr(), 0, 0)
        _lib.check(_lib.lib().spmm_route_backward(args, stream_handle(device)), 'route_topk_backward')
    return out


class _TopK(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, top, scoring, renormalize, scale, bias):
        out = _topk(logits, top, scoring, renormalize, scale, bias)
        ctx.save_for_backward(logits, out[1])
        ctx.how = (scoring, renormalize, scale)
        ctx.mark_non_differentiable(*out[1:])
        ctx.set_materialize_grads(False)      # or the routing would come back as four tensors of zeros
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dweights, *_):
        logits, experts = ctx.saved_tensors
        if dweights is None:
            return (None,) * 6
        return _topk_backward(dweights, logits, experts, *ctx.how), None, None, None, None, None


def route_topk(logits: torch.Tensor, top: int, *, scoring: str = 'softmax', renormalize: bool = True,
               scale: float = 1.0, bias: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Routing]:
    """Each token's ``top`` experts, their weights, and the rows grouped by expert.

    ``logits`` [T, E] (float32, bfloat16 or float16; E <= 1024, top <= 32).  The
    experts with the largest ``float32(logit) + bias`` are chosen, best first,
    ties to the lowest index; an expert whose logit is -inf or NaN is never
    chosen, and a token without any left gets expert -1 with weight 0, so a
    masked row takes no part.  ``bias`` [E] float32 moves the choice only; it is
    added to the logit with either scoring.  A router whose bias is added to the
    sigmoid chooses other experts and is not this one.

    The weights [T, top] float32 are the chosen experts' softmax over all E
    logits (or their sigmoid), divided by their sum over the chosen ones with
    ``renormalize``, times ``scale``; a renormalised sigmoid whose logit is below
    -709 (the type's lowest value as a mask) counts as 0.  Differentiable in
    ``logits``.
    """
    _check_score(logits, scoring)
    tokens, experts = logits.shape
    if isinstance(top, bool) or not isinstance(top, int) or top < 1 or top > experts:
        raise ValueError(f'top must be an integer in [1, {experts}]')
    if experts > _lib.MAX_GROUPS or top > _lib.MAX_TOP or tokens * top > 2**31 - 1:
        raise ValueError(f'route_topk takes up to {_lib.MAX_GROUPS} experts, {_lib.MAX_TOP} choices and 2**31 - 1 rows')
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (experts,)
                             or bias.device != logits.device):
        raise ValueError(f'bias must be a float32 tensor of {experts} values on the logits\' device')
    if forward_ad._current_level >= 0:
        refuse_tangents(logits=logits)
    need_cuda(logits, 'logits')
    bias = None if bias is None else bias.detach().contiguous()
    if logits.requires_grad and torch.is_grad_enabled():
        out = _TopK.apply(logits, top, scoring, renormalize, float(scale), bias)
    else:
        out = _topk(logits, top, scoring, renormalize, float(scale), bias)
    return out[0], Routing(*out[1:])


def route_topk_backward(dweights: torch.Tensor, logits: torch.Tensor, routing: Routing, *,
                        scoring: str = 'softmax', renormalize: bool = True, scale: float = 1.0) -> torch.Tensor:
    """Gradient of ``route_topk``'s weights with respect to ``logits`` (what autograd calls)."""
    _check_score(logits, scoring)
    check_routing(routing, logits.device)
    if routing.tokens != logits.shape[0] or routing.num_experts != logits.shape[1]:
        raise ValueError('routing does not belong to these logits')
    if dweights.shape != routing.slots.shape or dweights.dtype != torch.float32 or dweights.device != logits.device:
        raise ValueError('dweights must be float32, of the weights\' shape and on their device')
    if forward_ad._current_level >= 0:
        refuse_tangents(dweights=dweights, logits=logits)
    need_cuda(logits, 'logits')
    return _topk_backward(dweights, logits, routing.experts, scoring, renormalize, float(scale))


def _combine(y, routing, weights, residual):
    y, weights = _unit_rows(y), weights.contiguous()
    slots, n = routing.slots, y.shape[1]
    tokens, top = slots.shape
    with on_device(y.device):
        out = y.new_empty((tokens, n))
        res, res_ld = 0, 0
        if residual is not None:
            residual = _unit_rows(residual)
            res, res_ld = residual.data_ptr(), residual.stride(0)
        args = _COMBINE(1, _TYPES[y.dtype], tokens, top, y.shape[0], n, routing.num_experts, slots.data_ptr(),
                        routing.offsets.data_ptr(), weights.data_ptr(), y.data_ptr(), res, out.data_ptr(), 0, 0, 0,
                        y.stride(0), res_ld, n, 0, 0)
        _lib.check(_lib.lib().spmm_combine(args, stream_handle(y.device)), 'route_combine')
    return out


def _combine_backward(dout, y, slots, offsets, rows, weights, need_dy=True, need_dweights=True):
    y, dout, weights = _unit_rows(y), _unit_rows(dout), weights.contiguous()
    n = y.shape[1]
    with on_device(y.device):
        dy = y.new_empty(y.shape) if need_dy else None
        dw = weights.new_empty(weights.shape) if need_dweights else None
        args = _COMBINE(1, _TYPES[y.dtype], *slots.shape, y.shape[0], n, offsets.shape[0] - 1, slots.data_ptr(),
                        offsets.data_ptr(), weights.data_ptr(), y.data_ptr(), 0, 0, dout.data_ptr(),
                        dy.data_ptr() if need_dy else 0, dw.data_ptr() if need_dweights else 0, y.stride(0), 0, 0,
                        dout.stride(0), n)
        _lib.check(_lib.lib().spmm_combine_backward_rows(args, rows.data_ptr(), stream_handle(y.device)),
                   'route_combine_backward')
    return dy, dw


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, residual, routing):
        # the routing too, so that writing it again before the backward pass is an error
        ctx.save_for_backward(y, weights, routing.slots, routing.offsets, routing.rows)
        ctx.has_residual = residual is not None
        ctx.set_materialize_grads(False)
        return _combine(y, routing, weights, residual)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        y, weights, *routing = ctx.saved_tensors
        need = ctx.needs_input_grad
        dy = dw = None
        if dout is not None and (need[0] or need[1]):
            dy, dw = _combine_backward(dout, y, *routing, weights, need[0], need[1])
        return dy, dw, dout if ctx.has_residual and need[2] else None, None


def _check_combine(y, routing, weights):
    if y.dim() != 2 or y.layout != torch.strided:
        raise ValueError(f'y must be a dense 2D tensor, got {y.dim()}D')
    if y.dtype not in _TYPES:
        raise TypeError(f'y must be float32, bfloat16 or float16, got {y.dtype}')
    check_routing(routing, y.device)
    if y.numel() >= 2**31 - 1024 and max(y.shape) >= 2**31 - 1024:
        raise ValueError('y must have less than 2**31 - 1024 rows and columns')
    if y.shape[0] != routing.rows.shape[0]:
        raise ValueError(f'y has {y.shape[0]} rows, the routing {routing.rows.shape[0]}')
    if weights.shape != routing.slots.shape or weights.dtype != torch.float32 or weights.device != y.device:
        raise ValueError('weights must be float32, of the routing\'s shape and on y\'s device')


def route_combine(y: torch.Tensor, routing: Routing, weights: torch.Tensor,
                  residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out[t] = sum_j weights[t, j] * y[slots[t, j]] + residual[t]``, [T, N] in y's type.

    ``y`` [T*k, N] holds the grouped rows (``grouped_matmul``); choices without
    a slot add nothing.  Sums in float32 in the order of j, one rounding.
    Differentiable in ``y``, ``weights`` and ``residual``.
    """
    _check_combine(y, routing, weights)
    shape = (routing.tokens, y.shape[1])
    if residual is not None and (residual.shape != shape or residual.dtype != y.dtype
                                 or residual.device != y.device):
        raise ValueError(f'residual must be {shape} of y\'s type on its device')
    if forward_ad._current_level >= 0:
        refuse_tangents(y=y, weights=weights, residual=residual)
    need_cuda(y, 'y')
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (y, weights, residual)):
        return _Combine.apply(y, weights, residual, routing)
    return _combine(y, routing, weights, residual)


def route_combine_backward(dout: torch.Tensor, y: torch.Tensor, routing: Routing,
                           weights: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(dy, dweights) of ``route_combine`` (what autograd calls); the residual's gradient is ``dout``."""
    _check_combine(y, routing, weights)
    if dout.shape != (routing.tokens, y.shape[1]) or dout.dtype != y.dtype or dout.device != y.device:
        raise ValueError('dout must have the result\'s shape, type and device')
    if forward_ad._current_level >= 0:
        refuse_tangents(dout=dout, y=y, weights=weights)
    need_cuda(y, 'y')
    return _combine_backward(dout, y, routing.slots, routing.offsets, routing.rows, weights)
