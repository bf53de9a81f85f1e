"""Dense, grouped and routed products: refusals that need no GPU."""

import pytest
import torch
from torch.autograd import forward_ad

import spmm_b200 as S

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
