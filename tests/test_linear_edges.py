"""Dense, grouped and routed products: refusals that need no GPU."""

import ctypes as C

import pytest
import torch
from torch.autograd import forward_ad

import spmm_b200 as S
from spmm_b200 import _lib

BF = torch.bfloat16


def rand(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


def routing(t=4, k=2, e=3):
    return S.Routing(torch.zeros(t, k, dtype=torch.int32), torch.zeros(t, k, dtype=torch.int32),
                     torch.zeros(t * k, dtype=torch.int32), torch.zeros(e + 1, dtype=torch.int32))


def dual(*shape, dtype=BF):
    return forward_ad.make_dual(rand(*shape, dtype=dtype), torch.ones(*shape, dtype=dtype))


@pytest.mark.parametrize('call', [
    lambda: S.dense_matmul(dual(4, 8), rand(8, 6)),
    lambda: S.dense_matmul(rand(4, 8), dual(8, 6)),
    lambda: S.dense_matmul(rand(4, 8), rand(8, 6), dual(6)),
    lambda: S.dense_matmul(rand(4, 8), rand(8, 6), None, dual(4, 6)),
    lambda: S.dense_matmul_backward(dual(4, 6), rand(4, 8), rand(8, 6)),
    lambda: S.grouped_matmul(dual(8, 8), rand(3, 8, 6), routing()),
    lambda: S.grouped_matmul_backward(dual(8, 6), rand(8, 8), rand(3, 8, 6), routing()),
    lambda: S.route_topk(dual(4, 3, dtype=torch.float32), 2),
    lambda: S.route_topk_backward(dual(4, 2, dtype=torch.float32), rand(4, 3), routing()),
    lambda: S.route_combine(dual(8, 6), routing(), rand(4, 2, dtype=torch.float32)),
    lambda: S.route_combine(rand(8, 6), routing(), dual(4, 2, dtype=torch.float32)),
    lambda: S.route_combine(rand(8, 6), routing(), rand(4, 2, dtype=torch.float32), dual(4, 6)),
    lambda: S.route_combine_backward(dual(4, 6), rand(8, 6), routing(), rand(4, 2, dtype=torch.float32)),
])
def test_tangents_are_refused(call):
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match='tangent'):
        call()


def many(*shape):
    """A tensor of any size in one element."""
    return torch.zeros(1, dtype=BF).expand(*shape)


@pytest.mark.parametrize('call', [
    lambda: S.dense_matmul(many(2**31, 8), rand(8, 6)),
    lambda: S.dense_matmul(many(2**16, 2**15, 8), rand(8, 6)),
    lambda: S.dense_matmul(rand(4, 8), many(8, 2**31)),
    lambda: S.dense_matmul(many(4, 2**31), many(2**31, 8)),
    lambda: S.dense_matmul_backward(many(4, 2**31), rand(4, 8), many(8, 2**31)),
    lambda: S.grouped_matmul(rand(8, 8), many(3, 8, 2**31), torch.zeros(4, dtype=torch.int32)),
    lambda: S.route_combine(many(8, 2**31), routing(), torch.zeros(4, 2)),
    lambda: S.route_combine_backward(many(4, 2**31 - 1024), many(8, 2**31 - 1024), routing(), torch.zeros(4, 2)),
])
def test_sizes_past_the_limit_are_refused(call):
    with pytest.raises(ValueError, match=r'below 2\*\*31|less than 2\*\*31'):
        call()


def linear(**kw):
    """100 rows of bias gradients: what needs a workspace and no device to be refused."""
    a = _lib.Linear()
    a.version, a.dtype, a.groups, a.rows, a.x_rows, a.k, a.n = 1, _lib.DENSE_BF16, 1, 100, 100, 8, 8
    a.x_ld = a.w_k = a.y_ld = a.dy_ld = a.dx_ld = a.dw_k = a.dbias_g = 8
    a.w_n = a.dw_n = 1
    for name, v in dict(dy=256, dbias=256, workspace=256, workspace_bytes=1 << 20).items():
        setattr(a, name, v)
    for name, v in kw.items():
        setattr(a, name, v)
    return a


@pytest.mark.parametrize('field, value', [('workspace', 384), ('workspace', 264), ('x', 257), ('w', 257), ('dy', 257),
                                          ('dbias', 257), ('slope', 257), ('dx', 257), ('dw', 257), ('offsets', 258),
                                          ('gather', 258), ('slots', 258), ('status', 258), ('y', 257),
                                          ('residual', 257), ('bias', 257)])
def test_misaligned_pointers_of_a_product(field, value):
    L, a = _lib.lib(), linear(**{field: value})
    assert L.spmm_linear_backward(C.byref(a), None) == _lib.SPMM_EALIGN
    assert L.spmm_linear_forward(C.byref(a), None) == _lib.SPMM_EALIGN


@pytest.mark.parametrize('field, value', [('workspace', 264), ('logits', 258), ('weights', 258), ('experts_out', 257),
                                          ('slots', 258), ('rows', 258), ('offsets', 258), ('bias', 258),
                                          ('dweights', 258), ('dlogits', 258)])
def test_misaligned_pointers_of_a_routing(field, value):
    a = _lib.RouteArgs()
    a.version, a.dtype, a.tokens, a.experts, a.top, a.logits_ld = 1, _lib.DENSE_F32, 1000, 64, 4, 64
    for name in ('logits', 'weights', 'experts_out', 'slots', 'rows', 'offsets', 'dweights', 'dlogits', 'workspace'):
        setattr(a, name, 256)
    a.workspace_bytes = 1 << 20
    setattr(a, field, value)
    assert _lib.lib().spmm_route(C.byref(a), None) == _lib.SPMM_EALIGN
    assert _lib.lib().spmm_route_backward(C.byref(a), None) == _lib.SPMM_EALIGN


@pytest.mark.parametrize('field, value', [('y', 257), ('residual', 257), ('out', 257), ('dout', 257), ('dy', 257),
                                          ('slots', 258), ('offsets', 258), ('weights', 258), ('dweights', 258)])
def test_misaligned_pointers_of_a_combination(field, value):
    a = _lib.CombineArgs()
    a.version, a.dtype, a.tokens, a.top, a.rows, a.n, a.experts = 1, _lib.DENSE_BF16, 4, 2, 8, 8, 3
    a.y_ld = a.residual_ld = a.out_ld = a.dout_ld = a.dy_ld = 8
    for name in ('slots', 'offsets', 'weights', 'y', 'out', 'dout', 'dy', 'dweights'):
        setattr(a, name, 256)
    L = _lib.lib()
    assert L.spmm_combine_backward_rows(C.byref(a), 258, None) == _lib.SPMM_EALIGN
    setattr(a, field, value)
    for run in (L.spmm_combine, L.spmm_combine_backward):
        assert run(C.byref(a), None) == _lib.SPMM_EALIGN
