"""Dense and grouped products of 16-bit operands.

``dense_matmul``: ``y = act(x @ w + bias) + residual``.  ``grouped_matmul``: the
same for ragged groups of rows, each with a dense block of its own -- a
block-diagonal matrix with ragged blocks, the products of a mixture of experts.
Both are differentiable; ``dense_matmul_backward`` / ``grouped_matmul_backward``
are the gradients as plain calls.  Not in the reference.

Operands are bfloat16 or float16, sums float32, every output is rounded once.
No call waits for the GPU; like ``boo_matmul``'s, a result carries the status
of its bounded device waits (``product_status(y)``, ``check_product(y)``).
"""

from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple, Union

import torch

from . import _lib
from ._device import on_device, ptr, stream_handle
from .route import Routing, check_routing, need_cuda

__all__ = ['dense_matmul', 'dense_matmul_backward', 'grouped_matmul', 'grouped_matmul_backward', 'ACTIVATIONS']

ACTIVATIONS = ('none', 'relu', 'gelu', 'gelu_tanh', 'silu')
_TYPES = {torch.bfloat16: _lib.DENSE_BF16, torch.float16: _lib.DENSE_F16}


def _unit_rows(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _w_strides(w: torch.Tensor) -> Tuple[torch.Tensor, int, int]:
    """(w [G,K,N] with unit stride along k or n, the two strides)."""
    k, n = w.shape[1], w.shape[2]
    if w.stride(2) == 1 or n <= 1:
        return w, w.stride(1) if k > 1 else max(n, 1), 1
    if w.stride(1) == 1 or k <= 1:
        return w, 1, w.stride(2) if n > 1 else max(k, 1)
    w = w.contiguous()
    return w, w.stride(1), 1


class _Groups:
    """The grouping as the C entries take it."""

    __slots__ = ('offsets', 'gather', 'slots', 'rows', 'count')

    def __init__(self, offsets, gather, slots, rows, count):
        self.offsets, self.gather, self.slots, self.rows, self.count = offsets, gather, slots, rows, count


def _struct(x, w, g):
    """spmm_linear with everything both directions share (x [R,K] and w [G,K,N] prepared)."""
    w, sk, sn = _w_strides(w)
    a = _lib.Linear()
    a.version, a.dtype = 1, _TYPES[x.dtype]
    a.rows, a.k, a.n, a.groups, a.x_rows = g.rows, w.shape[1], w.shape[2], g.count, x.shape[0]
    a.offsets, a.gather = ptr(g.offsets), ptr(g.gather)
    if g.slots is not None:
        a.slots, a.top = ptr(g.slots), g.slots.shape[1]
    a.x, a.x_ld = ptr(x), x.stride(0)
    a.w, a.w_k, a.w_n, a.w_g = ptr(w), sk, sn, w.stride(0)
    return a, w


def _scratch(a, size, device):
    n = (size + 255) // 256 * 256
    buf = torch.empty(n + 256, dtype=torch.uint8, device=device)
    p = buf.data_ptr()
    a.workspace, a.workspace_bytes, a.status = p if size else None, size, p + n
    return buf, buf[n:n + 4].view(torch.int32)


def _forward(x, w, g, bias, residual, activation, want_slope):
    device = x.device
    x = _unit_rows(x)
    a, w = _struct(x, w, g)
    a.activation = ACTIVATIONS.index(activation)
    L = _lib.lib()
    with on_device(device):
        y = torch.empty((g.rows, w.shape[2]), dtype=x.dtype, device=device)
        a.y, a.y_ld = ptr(y), y.stride(0)
        if bias is not None:
            bias = _unit_rows(bias)
            a.bias, a.bias_g = ptr(bias), bias.stride(0)
        if residual is not None:
            residual = _unit_rows(residual)
            a.residual, a.residual_ld = ptr(residual), residual.stride(0)
        slope = None
        if want_slope and activation != 'none':
            slope = torch.empty(y.shape, dtype=torch.int16, device=device)
            a.slope = ptr(slope)
        keep, status = _scratch(a, L.spmm_linear_forward_workspace_size(C.byref(a)), device)
        _lib.check(L.spmm_linear_forward(C.byref(a), stream_handle(device)), 'matmul')
        del keep
    return y, slope, status


def _backward(dy, x, w, g, slope, need_dx, need_dw, need_dbias):
    device = x.device
    x, dy = _unit_rows(x), _unit_rows(dy)
    a, w = _struct(x, w, g)
    L = _lib.lib()
    with on_device(device):
        a.dy, a.dy_ld = ptr(dy), dy.stride(0)
        a.slope = ptr(slope)
        dx = dw = dbias = None
        if need_dx:
            dx = torch.empty(x.shape, dtype=x.dtype, device=device)
            a.dx, a.dx_ld = ptr(dx), dx.stride(0)
        if need_dw:
            count, k, n = w.shape
            if a.w_n == 1:
                dw = torch.empty((count, k, n), dtype=x.dtype, device=device)
                a.dw_k, a.dw_n = max(n, 1), 1
            else:
                dw = torch.empty((count, n, k), dtype=x.dtype, device=device).transpose(1, 2)
                a.dw_k, a.dw_n = 1, max(k, 1)
            a.dw, a.dw_g = ptr(dw), k * n
        if need_dbias:
            dbias = torch.empty((g.count, w.shape[2]), dtype=x.dtype, device=device)
            a.dbias, a.dbias_g = ptr(dbias), dbias.stride(0)
        keep, status = _scratch(a, L.spmm_linear_backward_workspace_size(C.byref(a)), device)
        _lib.check(L.spmm_linear_backward(C.byref(a), stream_handle(device)), 'matmul_backward')
        del keep
    for t in (dx, dw, dbias):
        if t is not None:
            t._spmm_status = status
    return dx, dw, dbias


class _MatMul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, residual, activation, g):
        y, slope, status = _forward(x, w, g, bias, residual, activation, True)
        ctx.save_for_backward(x, w, slope)
        ctx.g = g
        ctx.mark_non_differentiable(status)
        return y, status

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, _):
        x, w, slope = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = dw = db = None
        if need[0] or need[1] or need[2]:
            dx, dw, db = _backward(dy, x, w, ctx.g, slope, need[0], need[1], need[2])
        return dx, dw, db, dy if need[3] else None, None, None


def _check_xw(x, w, w_dim):
    for name, t in (('x', x), ('w', w)):
        if not isinstance(t, torch.Tensor) or t.layout != torch.strided:
            raise ValueError(f'{name} must be a dense tensor')
    if w.dim() != w_dim:
        raise ValueError(f'Expected {w_dim}D w, got {w.dim()}D')
    if x.dtype not in _TYPES:
        raise TypeError(f'x must be bfloat16 or float16, got {x.dtype}')
    if w.dtype != x.dtype:
        raise TypeError(f'w dtype must match x ({x.dtype}), got {w.dtype}')
    if x.dim() < 1 or x.shape[-1] != w.shape[-2]:
        raise ValueError(f'x has {x.shape[-1] if x.dim() else 0} columns, expected {w.shape[-2]}')
    if w.device != x.device:
        raise ValueError('w must be on x\'s device')


def _check_like(name, t, x, shape):
    if t.shape != shape or t.layout != torch.strided:
        raise ValueError(f'{name} must be {tuple(shape)}, got {tuple(t.shape)}')
    if t.dtype != x.dtype:
        raise TypeError(f'{name} dtype must match x ({x.dtype}), got {t.dtype}')
    if t.device != x.device:
        raise ValueError(f'{name} must be on x\'s device')


def _check_slope(slope, shape, x):
    if slope is not None and (slope.shape != shape or slope.dtype != torch.int16 or not slope.is_contiguous()
                              or slope.device != x.device):
        raise ValueError('slope must be what the forward call returned')


def _run(x, w, g, bias, residual, activation, return_slope):
    if return_slope:
        y, slope, status = _forward(x, w, g, bias, residual, activation, True)
        y._spmm_status = status
        return y, slope
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, w, bias, residual)):
        y, status = _MatMul.apply(x, w, bias, residual, activation, g)
    else:
        y, _, status = _forward(x, w, g, bias, residual, activation, False)
    y._spmm_status = status
    return y


def dense_matmul(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None,
                 residual: Optional[torch.Tensor] = None, *, activation: str = 'none',
                 return_slope: bool = False):
    """``act(x @ w + bias) + residual``: x [..., K], w [K, N], bias [N], residual [..., N].

    bfloat16 or float16, the same for every operand; sums in float32, one
    rounding.  ``w`` may have unit stride along either dimension (``weight.t()``
    of an [N, K] weight costs no copy).  Differentiable; inside a CUDA graph
    capture use ``return_slope=True`` and ``dense_matmul_backward``, which
    involve no autograd graph: ``(y, slope)`` comes back, ``slope`` (int16
    fixed point, None without an activation) being the activation's derivative.
    """
    if activation not in ACTIVATIONS:
        raise ValueError(f'activation must be one of {ACTIVATIONS}')
    _check_xw(x, w, 2)
    shape = x.shape[:-1] + (w.shape[1],)
    if bias is not None:
        _check_like('bias', bias, x, (w.shape[1],))
    if residual is not None:
        _check_like('residual', residual, x, shape)
    need_cuda(x, 'x')
    x2 = x.reshape(_rows(x), x.shape[-1])
    res = None if residual is None else residual.reshape(x2.shape[0], w.shape[1])
    g = _Groups(None, None, None, x2.shape[0], 1)
    out = _run(x2, w.unsqueeze(0), g, None if bias is None else bias.unsqueeze(0), res, activation, return_slope)
    if x.dim() == 2:
        return out
    y = out[0] if return_slope else out
    status = y._spmm_status
    y = y.reshape(shape)
    y._spmm_status = status
    return (y, out[1]) if return_slope else y


def _rows(x: torch.Tensor) -> int:
    n = 1
    for s in x.shape[:-1]:
        n *= s
    return n


def dense_matmul_backward(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor, slope: Optional[torch.Tensor] = None,
                          *, bias: bool = False):
    """(dx, dw, dbias) of ``dense_matmul`` given ``slope`` of its forward call; dbias is None unless ``bias``.

    The residual's gradient is ``dy``.  ``dy * act'`` is rounded to the operands'
    type for the two products.
    """
    _check_xw(x, w, 2)
    shape = x.shape[:-1] + (w.shape[1],)
    _check_like('dy', dy, x, shape)
    rows = _rows(x)
    _check_slope(slope, (rows, w.shape[1]), x)
    need_cuda(x, 'x')
    g = _Groups(None, None, None, rows, 1)
    x2 = x.reshape(rows, x.shape[-1])
    dx, dw, db = _backward(dy.reshape(rows, w.shape[1]), x2, w.unsqueeze(0), g, slope, True, True, bias)
    status = dx._spmm_status
    dx, dw = dx.reshape(x.shape), dw.squeeze(0)
    dx._spmm_status = dw._spmm_status = status
    return dx, dw, None if db is None else db.squeeze(0)


def _groups(x, w, groups, gather):
    if isinstance(groups, Routing):
        check_routing(groups, x.device)
        offsets, rows = groups.offsets, groups.rows.shape[0]
        if gather:
            if x.shape[0] != groups.tokens:
                raise ValueError(f'x has {x.shape[0]} rows, the routing {groups.tokens} tokens')
        elif x.shape[0] != rows:
            raise ValueError(f'x has {x.shape[0]} rows, the routing {rows}')
    else:
        offsets, rows = groups, x.shape[0]
        if not isinstance(offsets, torch.Tensor) or offsets.dtype != torch.int32 or offsets.dim() != 1 \
                or not offsets.is_contiguous():
            raise ValueError('groups must be a Routing or a contiguous 1D int32 tensor of offsets')
        if gather:
            raise ValueError('gather=True needs a Routing')
        if offsets.device != x.device:
            raise ValueError('groups must be on x\'s device')
    count = offsets.shape[0] - 1
    if count != w.shape[0]:
        raise ValueError(f'{count} groups, but w holds {w.shape[0]} blocks')
    if not 1 <= count <= _lib.MAX_GROUPS:
        raise ValueError(f'grouped_matmul takes 1 to {_lib.MAX_GROUPS} groups, got {count}')
    return _Groups(offsets, groups.rows if gather else None, groups.slots if gather else None, rows, count)


def grouped_matmul(x: torch.Tensor, w: torch.Tensor, groups: Union[Routing, torch.Tensor],
                   bias: Optional[torch.Tensor] = None, *, activation: str = 'none', gather: bool = False,
                   return_slope: bool = False):
    """``y[r] = act(x[r] @ w[g] + bias[g])`` for the rows r of each group g; w [G, K, N], bias [G, N].

    ``groups``: a ``Routing``, or int32 offsets [G+1] on the device (offsets[0] =
    0, non-decreasing): group g owns rows offsets[g] .. offsets[g+1].  Rows
    behind the last group are zero.  With ``gather`` (a ``Routing``) x holds the
    tokens [T, K] and row r reads token ``rows[r]``; without it x is [R, K] in
    grouped order.  Types, strides of w, differentiation and ``return_slope``
    as in ``dense_matmul``.  Offsets are read on the device and cannot be
    checked here: a table that decreases or leaves [0, R] gives wrong values,
    but reads and writes nothing outside the operands.
    """
    if activation not in ACTIVATIONS:
        raise ValueError(f'activation must be one of {ACTIVATIONS}')
    _check_xw(x, w, 3)
    if x.dim() != 2:
        raise ValueError(f'Expected 2D x, got {x.dim()}D')
    g = _groups(x, w, groups, gather)
    if bias is not None:
        _check_like('bias', bias, x, (w.shape[0], w.shape[2]))
    need_cuda(x, 'x')
    return _run(x, w, g, bias, None, activation, return_slope)


def grouped_matmul_backward(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor,
                            groups: Union[Routing, torch.Tensor], slope: Optional[torch.Tensor] = None, *,
                            gather: bool = False, bias: bool = False):
    """(dx, dw, dbias) of ``grouped_matmul``; dbias is None unless ``bias``.

    Empty groups get zeros, rows behind the last group a zero dx.  With
    ``gather`` dx [T, K] sums over the rows that read the token, in float32.
    """
    _check_xw(x, w, 3)
    if x.dim() != 2:
        raise ValueError(f'Expected 2D x, got {x.dim()}D')
    g = _groups(x, w, groups, gather)
    _check_like('dy', dy, x, (g.rows, w.shape[2]))
    _check_slope(slope, (g.rows, w.shape[2]), x)
    need_cuda(x, 'x')
    return _backward(dy, x, w, g, slope, True, True, bias)
