"""Dense and grouped products of 16-bit operands.

``dense_matmul``: ``y = act(x @ w + bias) + residual``.  ``grouped_matmul``: the
same for ragged groups of rows, each with a dense block of its own -- a
block-diagonal matrix with ragged blocks, the products of a mixture of experts.
Both are differentiable; ``dense_matmul_backward`` / ``grouped_matmul_backward``
are the gradients as plain calls.  Not in the reference.

Operands are bfloat16 or float16, sums float32.  Every output is rounded once;
dx and dw come from ``dz = dy * act'(z)``, which is rounded to the operands'
type before (not without an activation).
No call waits for the GPU; like ``boo_matmul``'s, a result carries the status
of its bounded device waits (``product_status(y)``, ``check_product(y)``), and
after a backward pass through autograd that of its gradients' waits as well.
"""

from __future__ import annotations

import ctypes as C
import struct
from typing import Optional, Tuple, Union

import torch
from torch.autograd import forward_ad

from . import _lib
from ._device import on_device, stream_handle
from .route import Routing, check_routing, need_cuda, refuse_tangents

__all__ = ['dense_matmul', 'dense_matmul_backward', 'grouped_matmul', 'grouped_matmul_backward', 'ACTIVATIONS']

ACTIVATIONS = ('none', 'relu', 'gelu', 'gelu_tanh', 'silu')
_ACT = {name: i for i, name in enumerate(ACTIVATIONS)}
_TYPES = {torch.bfloat16: _lib.DENSE_BF16, torch.float16: _lib.DENSE_F16}


# spmm_linear (include/spmm_b200.h) packed in one go: filling a ctypes structure field by field cost as much
# host time as launching the product
_PACK = struct.Struct('@6i5q3Pq10P13qPQP').pack
assert struct.calcsize('@6i5q3Pq10P13qPQP') == C.sizeof(_lib.Linear)


def _unit_rows(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _w_strides(w: torch.Tensor):
    """(w [..., K, N] with unit stride along k or n, the strides along k, n and the groups)."""
    k, n = w.shape[-2], w.shape[-1]
    st = w.stride()
    if st[-1] != 1 and n > 1 and st[-2] != 1 and k > 1:
        w = w.contiguous()
        st = w.stride()
    sg = st[0] if len(st) == 3 else 0
    if st[-1] == 1 or n <= 1:
        return w, (st[-2] if k > 1 else max(n, 1), 1, sg)
    return w, (1, st[-1] if n > 1 else max(k, 1), sg)


class _Groups:
    """The grouping as the C entries take it."""

    __slots__ = ('offsets', 'gather', 'slots', 'rows', 'count')

    def __init__(self, offsets, gather, slots, rows, count):
        self.offsets, self.gather, self.slots, self.rows, self.count = offsets, gather, slots, rows, count

    def pointers(self):
        """offsets, gather, slots, top."""
        if self.offsets is None:
            return 0, 0, 0, 0
        if self.gather is None:
            return self.offsets.data_ptr(), 0, 0, 0
        return self.offsets.data_ptr(), self.gather.data_ptr(), self.slots.data_ptr(), self.slots.shape[1]


def _call(name, fixed, x, where, scratch, word=None):
    """Runs a C entry on x's device and stream; returns the call's status word (`word`, or a new one).  Where `scratch` says that a
    workspace is likely its size is asked for first; a call that needs one after all says so before it does
    anything and is repeated with it."""
    L = _lib.lib()
    run = getattr(L, name)
    stream = stream_handle(x.device)
    if word is None:
        word = x.new_empty(2)                   # 4 bytes
    rc = _lib.SPMM_EWORKSPACE
    if not scratch:
        rc = run(_PACK(*fixed, 0, 0, word.data_ptr()), stream)
    if rc == _lib.SPMM_EWORKSPACE:
        n = getattr(L, name + '_workspace_size')(_PACK(*fixed, 0, 0, 0))
        ws = torch.empty(n, dtype=torch.uint8, device=x.device) if n else None
        rc = run(_PACK(*fixed, ws.data_ptr() if n else 0, n, word.data_ptr()), stream)
    if rc:
        _lib.check(rc, where)
    return word


def _forward(x, w, g, bias, residual, activation, want_slope):
    """x [rows, K], w [K,N] or [G,K,N], bias [N] or [G,N], residual [rows, N]."""
    x = _unit_rows(x)
    w, (sk, sn, sg) = _w_strides(w)
    k, n = w.shape[-2:]
    rows = g.rows
    with on_device(x.device):
        y = x.new_empty((rows, n))
        slope = None
        if want_slope and activation != 'none':
            slope = torch.empty((rows, n), dtype=torch.int16, device=x.device)
        bias_g = res_ld = 0
        if bias is not None:
            bias = _unit_rows(bias)
            bias_g = bias.stride(0) if bias.dim() == 2 else 0
        if residual is not None:
            residual = _unit_rows(residual)
            res_ld = residual.stride(0)
        status = _call('spmm_linear_forward', (
            1, _TYPES[x.dtype], _ACT[activation], 0, 0, 0, rows, k, n, g.count, x.shape[0], *g.pointers(),
            x.data_ptr(), w.data_ptr(), 0 if bias is None else bias.data_ptr(),
            0 if residual is None else residual.data_ptr(), y.data_ptr(), 0 if slope is None else slope.data_ptr(),
            0, 0, 0, 0, x.stride(0), sk, sn, sg, bias_g, res_ld, n, 0, 0, 0, 0, 0, 0), x, 'matmul',
            (k | (n if sn == 1 else 0)) % 8 != 0)
    return y, slope, status


def _backward(dy, x, x_rows, w, g, slope, need_dx, need_dw, need_dbias, word=None):
    """x is needed for dw alone, None without it.  `word`: a status word that keeps what it says already."""
    dy = _unit_rows(dy)
    w, (sk, sn, sg) = _w_strides(w)
    k, n = w.shape[-2:]
    x_ptr, x_ld = 0, k
    if x is not None:
        x = _unit_rows(x)
        x_ptr, x_ld = x.data_ptr(), x.stride(0)
    with on_device(dy.device):
        dx = dw = dbias = None
        dw_k = dw_n = 0
        if need_dx:
            dx = dy.new_empty((x_rows, k))
        if need_dw:
            lead = w.shape[:-2]
            if sn == 1:
                dw = dy.new_empty(lead + (k, n))
                dw_k, dw_n = max(n, 1), 1
            else:
                dw = dy.new_empty(lead + (n, k)).transpose(-2, -1)
                dw_k, dw_n = 1, max(k, 1)
        if need_dbias:
            dbias = dy.new_empty(w.shape[:-2] + (n,))
        status = _call('spmm_linear_backward', (
            1, _TYPES[dy.dtype], 0, 0, 0 if word is None else _lib.LINEAR_KEEP_STATUS, 0, g.rows, k, n, g.count, x_rows, *g.pointers(),
            x_ptr, w.data_ptr(), 0, 0, 0, 0 if slope is None else slope.data_ptr(), dy.data_ptr(),
            0 if dx is None else dx.data_ptr(), 0 if dw is None else dw.data_ptr(),
            0 if dbias is None else dbias.data_ptr(), x_ld, sk, sn, sg, 0, 0, 0, dy.stride(0), k, dw_k, dw_n,
            k * n, n), dy, 'matmul_backward', slope is not None or g.gather is not None or (k | n) % 8 != 0,
            word)
    for t in (dx, dw, dbias):
        if t is not None:
            t._spmm_status = status
    return dx, dw, dbias


class _MatMul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, residual, activation, g):
        need = ctx.needs_input_grad
        y, slope, status = _forward(x, w, g, bias, residual, activation, need[0] or need[1] or need[2])
        # the grouping too, so that writing it again before the backward pass is an error
        ctx.save_for_backward(x if need[1] else None, w, slope, status, g.offsets, g.gather, g.slots)
        ctx.counts = g.rows, g.count
        ctx.x_rows = x.shape[0]
        ctx.mark_non_differentiable(status)
        ctx.set_materialize_grads(False)      # or the status would come back as a tensor of zeros
        return y, status

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, _):
        x, w, slope, status, *groups = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = dw = db = None
        if dy is not None and (need[0] or need[1] or need[2]):
            dx, dw, db = _backward(dy, x, ctx.x_rows, w, _Groups(*groups, *ctx.counts), slope, *need[:3],
                                   word=status)   # y speaks for its gradients too
        return dx, dw, db, dy if need[3] else None, None, None


def _check_xw(x, w, w_dim):
    for name, t in (('x', x), ('w', w)):
        if not isinstance(t, torch.Tensor) or t.layout is not torch.strided:
            raise ValueError(f'{name} must be a dense tensor')
    if w.dim() != w_dim:
        raise ValueError(f'Expected {w_dim}D w, got {w.dim()}D')
    if x.dtype not in _TYPES:
        raise TypeError(f'x must be bfloat16 or float16, got {x.dtype}')
    if w.dtype is not x.dtype:
        raise TypeError(f'w dtype must match x ({x.dtype}), got {w.dtype}')
    if x.dim() < 1 or x.shape[-1] != w.shape[-2]:
        raise ValueError(f'x has {x.shape[-1] if x.dim() else 0} columns, expected {w.shape[-2]}')
    if w.get_device() != x.get_device():
        raise ValueError('w must be on x\'s device')
    if x.numel() >= 2**31 or w.numel() >= 2**31:
        if max(w.shape) >= 2**31 or _rows(x) >= 2**31:
            raise ValueError('rows, columns and features must be below 2**31')


def _check_like(name, t, x, shape):
    if not isinstance(t, torch.Tensor) or t.shape != shape or t.layout is not torch.strided:
        raise ValueError(f'{name} must be a dense tensor of shape {tuple(shape)}')
    if t.dtype is not x.dtype:
        raise TypeError(f'{name} dtype must match x ({x.dtype}), got {t.dtype}')
    if t.get_device() != x.get_device():
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
    if torch.is_grad_enabled() and (x.requires_grad or w.requires_grad
                                    or (bias is not None and bias.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
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
    if activation not in _ACT:
        raise ValueError(f'activation must be one of {ACTIVATIONS}')
    _check_xw(x, w, 2)
    shape = x.shape[:-1] + (w.shape[1],)
    if bias is not None:
        _check_like('bias', bias, x, (w.shape[1],))
    if residual is not None:
        _check_like('residual', residual, x, shape)
    if forward_ad._current_level >= 0:
        refuse_tangents(x=x, w=w, bias=bias, residual=residual)
    need_cuda(x, 'x')
    if x.dim() == 2:
        return _run(x, w, _Groups(None, None, None, x.shape[0], 1), bias, residual, activation, return_slope)
    rows = _rows(x)
    out = _run(x.reshape(rows, x.shape[-1]), w, _Groups(None, None, None, rows, 1), bias,
               None if residual is None else residual.reshape(rows, w.shape[1]), activation, return_slope)
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
    if forward_ad._current_level >= 0:
        refuse_tangents(dy=dy, x=x, w=w)
    need_cuda(x, 'x')
    g = _Groups(None, None, None, rows, 1)
    if x.dim() == 2:
        return _backward(dy, x, x.shape[0], w, g, slope, True, True, bias)
    dx, dw, db = _backward(dy.reshape(rows, w.shape[1]), x.reshape(rows, x.shape[-1]), rows, w, g, slope, True, True,
                           bias)
    status = dx._spmm_status
    dx = dx.reshape(x.shape)
    dx._spmm_status = status
    return dx, dw, db


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
    checked here: the first one counts as 0, and a table that decreases or
    leaves [0, R] gives wrong values, but reads and writes nothing outside the
    operands.
    """
    if activation not in _ACT:
        raise ValueError(f'activation must be one of {ACTIVATIONS}')
    _check_xw(x, w, 3)
    if x.dim() != 2:
        raise ValueError(f'Expected 2D x, got {x.dim()}D')
    g = _groups(x, w, groups, gather)
    if bias is not None:
        _check_like('bias', bias, x, (w.shape[0], w.shape[2]))
    if forward_ad._current_level >= 0:
        refuse_tangents(x=x, w=w, bias=bias)
    need_cuda(x, 'x')
    return _run(x, w, g, bias, None, activation, return_slope)


def grouped_matmul_backward(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor,
                            groups: Union[Routing, torch.Tensor], slope: Optional[torch.Tensor] = None, *,
                            gather: bool = False, bias: bool = False):
    """(dx, dw, dbias) of ``grouped_matmul``; dbias is None unless ``bias``.

    Empty groups get zeros, rows behind the last group a zero dx.  With
    ``gather`` dx [T, K] sums over the rows that the token's ``slots`` name, in
    float32.
    """
    _check_xw(x, w, 3)
    if x.dim() != 2:
        raise ValueError(f'Expected 2D x, got {x.dim()}D')
    g = _groups(x, w, groups, gather)
    _check_like('dy', dy, x, (g.rows, w.shape[2]))
    _check_slope(slope, (g.rows, w.shape[2]), x)
    if forward_ad._current_level >= 0:
        refuse_tangents(dy=dy, x=x, w=w)
    need_cuda(x, 'x')
    return _backward(dy, x, x.shape[0], w, g, slope, True, True, bias)
