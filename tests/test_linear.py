"""Dense, grouped and routed products: argument checks and the C entries' refusals (no GPU)."""

import ctypes as C

import pytest
import torch

import spmm_b200 as S
from spmm_b200 import _lib

BF = torch.bfloat16


def rand(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


def routing(t=4, k=2, e=3):
    return S.Routing(torch.zeros(t, k, dtype=torch.int32), torch.zeros(t, k, dtype=torch.int32),
                     torch.zeros(t * k, dtype=torch.int32), torch.zeros(e + 1, dtype=torch.int32))


@pytest.mark.parametrize('call, exc, text', [
    (lambda: S.dense_matmul(rand(4, 8), rand(8, 6), activation='tanh'), ValueError, 'activation'),
    (lambda: S.dense_matmul(rand(4, 8), rand(7, 6)), ValueError, 'columns'),
    (lambda: S.dense_matmul(rand(4, 8), rand(1, 8, 6)), ValueError, '2D w'),
    (lambda: S.dense_matmul(rand(4, 8, dtype=torch.float32), rand(8, 6, dtype=torch.float32)), TypeError, 'bfloat16'),
    (lambda: S.dense_matmul(rand(4, 8), rand(8, 6, dtype=torch.float16)), TypeError, 'w dtype'),
    (lambda: S.dense_matmul(rand(4, 8), rand(8, 6), rand(5)), ValueError, 'bias'),
    (lambda: S.dense_matmul(rand(4, 8), rand(8, 6), None, rand(4, 5)), ValueError, 'residual'),
    (lambda: S.dense_matmul(rand(4, 8), rand(8, 6), None, rand(4, 6, dtype=torch.float32)), TypeError, 'residual'),
    (lambda: S.dense_matmul(rand(4, 8), rand(8, 6)), ValueError, 'CUDA tensor'),
    (lambda: S.dense_matmul(torch.zeros(4, 8).to_sparse(), rand(8, 6)), ValueError, 'dense'),
    (lambda: S.dense_matmul_backward(rand(4, 5), rand(4, 8), rand(8, 6)), ValueError, 'dy'),
    (lambda: S.dense_matmul_backward(rand(4, 6), rand(4, 8), rand(8, 6), rand(4, 6)), ValueError, 'slope'),
    (lambda: S.grouped_matmul(rand(8, 8), rand(3, 8, 6), torch.zeros(4)), ValueError, 'offsets'),
    (lambda: S.grouped_matmul(rand(8, 8), rand(3, 8, 6), torch.zeros(3, dtype=torch.int32)), ValueError, 'blocks'),
    (lambda: S.grouped_matmul(rand(8, 8), rand(3, 8, 6), torch.zeros(4, dtype=torch.int32), gather=True), ValueError,
     'Routing'),
    (lambda: S.grouped_matmul(rand(8, 8), rand(3, 8, 6), routing(), gather=True), ValueError, 'tokens'),
    (lambda: S.grouped_matmul(rand(7, 8), rand(3, 8, 6), routing()), ValueError, 'rows'),
    (lambda: S.grouped_matmul(rand(8, 8), rand(3, 8, 6), routing(), rand(3, 5)), ValueError, 'bias'),
    (lambda: S.grouped_matmul(rand(8, 8), rand(0, 8, 6), torch.zeros(1, dtype=torch.int32)), ValueError, 'groups'),
    (lambda: S.grouped_matmul(rand(8, 8), rand(1025, 8, 6), torch.zeros(1026, dtype=torch.int32)), ValueError,
     'groups'),
    (lambda: S.grouped_matmul(rand(8, 8), rand(3, 8, 6), routing()), ValueError, 'CUDA tensor'),
    (lambda: S.route_topk(torch.zeros(4, 8), 0), ValueError, 'top'),
    (lambda: S.route_topk(torch.zeros(4, 8), 9), ValueError, 'top'),
    (lambda: S.route_topk(torch.zeros(4, 8), 2.0), ValueError, 'top'),
    (lambda: S.route_topk(torch.zeros(4, 64), 33), ValueError, 'up to'),
    (lambda: S.route_topk(torch.zeros(4, 1025), 2), ValueError, 'up to'),
    (lambda: S.route_topk(torch.zeros(4), 2), ValueError, '2D'),
    (lambda: S.route_topk(torch.zeros(4, 8, dtype=torch.float64), 2), TypeError, 'float32'),
    (lambda: S.route_topk(torch.zeros(4, 8), 2, scoring='relu'), ValueError, 'scoring'),
    (lambda: S.route_topk(torch.zeros(4, 8), 2, bias=torch.zeros(7)), ValueError, 'bias'),
    (lambda: S.route_topk(torch.zeros(4, 8), 2), ValueError, 'CUDA tensor'),
    (lambda: S.route_topk_backward(torch.zeros(4, 2), torch.zeros(4, 4), routing()), ValueError, 'belong'),
    (lambda: S.route_combine(rand(8, 6), routing(), torch.zeros(4, 3)), ValueError, 'weights'),
    (lambda: S.route_combine(rand(7, 6), routing(), torch.zeros(4, 2)), ValueError, 'rows'),
    (lambda: S.route_combine(rand(8, 6), 'x', torch.zeros(4, 2)), TypeError, 'Routing'),
    (lambda: S.route_combine(rand(8, 6), routing(), torch.zeros(4, 2), rand(4, 5)), ValueError, 'residual'),
    (lambda: S.route_combine(rand(8, 6), routing(), torch.zeros(4, 2)), ValueError, 'CUDA tensor'),
    (lambda: S.route_combine_backward(rand(4, 5), rand(8, 6), routing(), torch.zeros(4, 2)), ValueError, 'dout'),
])
def test_refusals(call, exc, text):
    with pytest.raises(exc, match=text):
        call()


def linear(**kw):
    a = _lib.Linear()
    a.version, a.dtype, a.groups, a.w_k, a.w_n = 1, _lib.DENSE_BF16, 1, 8, 1
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize('fields, status', [
    (dict(version=2), _lib.SPMM_EINVAL),
    (dict(dtype=0), _lib.SPMM_EUNSUPPORTED),
    (dict(rows=-1, x_rows=-1), _lib.SPMM_EINVAL),
    (dict(groups=0), _lib.SPMM_EINVAL),
    (dict(groups=1025, offsets=8), _lib.SPMM_EUNSUPPORTED),
    (dict(groups=2), _lib.SPMM_EINVAL),                       # several groups need offsets
    (dict(rows=4, x_rows=5), _lib.SPMM_EINVAL),               # only a gather changes the row count
    (dict(wait_us=10), _lib.SPMM_EINVAL),
    (dict(w_k=2, w_n=2), _lib.SPMM_EUNSUPPORTED),
    (dict(rows=1 << 31, x_rows=1 << 31), _lib.SPMM_EUNSUPPORTED),
])
def test_linear_sizes_are_checked_on_the_host(fields, status):
    L, a = _lib.lib(), linear(**fields)
    assert L.spmm_linear_forward(C.byref(a), None) == status
    assert L.spmm_linear_backward(C.byref(a), None) == status
    assert L.spmm_linear_forward_workspace_size(C.byref(a)) == 0


def test_linear_null_operands():
    L = _lib.lib()
    assert L.spmm_linear_forward(None, None) == _lib.SPMM_EINVAL
    assert L.spmm_linear_forward(C.byref(linear(rows=4, x_rows=4, k=8, n=8)), None) == _lib.SPMM_EINVAL
    assert L.spmm_linear_forward(C.byref(linear(activation=9)), None) == _lib.SPMM_EINVAL
    assert L.spmm_linear_backward(C.byref(linear(rows=4, x_rows=4, k=8, n=8, dx=16)), None) == _lib.SPMM_EINVAL
    assert L.spmm_linear_backward(C.byref(linear(rows=4, x_rows=4, k=8, n=8, dy=16, dw=16)), None) == _lib.SPMM_EINVAL


def test_route_and_combine_entries():
    L = _lib.lib()
    for f in (L.spmm_route, L.spmm_route_backward, L.spmm_combine, L.spmm_combine_backward):
        assert f(None, None) == _lib.SPMM_EINVAL
    a = _lib.RouteArgs()
    a.version, a.tokens, a.experts, a.top = 1, 1000, 64, 4
    assert L.spmm_route(C.byref(a), None) == _lib.SPMM_EINVAL             # no outputs
    need = L.spmm_route_workspace_size(C.byref(a))
    assert need > 0
    a.logits = a.weights = a.experts_out = a.slots = a.rows = a.offsets = 256
    assert L.spmm_route(C.byref(a), None) == _lib.SPMM_EWORKSPACE
    a.top = 33
    assert L.spmm_route(C.byref(a), None) == _lib.SPMM_EUNSUPPORTED
    a.top = 65
    assert L.spmm_route(C.byref(a), None) == _lib.SPMM_EINVAL
    c = _lib.CombineArgs()
    c.version, c.dtype, c.tokens, c.top, c.rows, c.n = 1, _lib.DENSE_BF16, 4, 2, 8, 8
    assert L.spmm_combine(C.byref(c), None) == _lib.SPMM_EINVAL
    c.dtype = 1
    assert L.spmm_combine(C.byref(c), None) == _lib.SPMM_EUNSUPPORTED


def test_struct_sizes_match_the_header():
    assert C.sizeof(_lib.Linear) == 6 * 4 + 8 * (5 + 3 + 1 + 10 + 13 + 3)
    assert C.sizeof(_lib.RouteArgs) == 4 * 4 + 8 * 3 + 8 * 3 + 8 + 8 * 8 + 8
    assert C.sizeof(_lib.CombineArgs) == 8 + 8 * 5 + 8 * 9 + 8 * 5
