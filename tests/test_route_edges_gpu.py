"""Expert choice and combination at the edges: logits far from 0, routings of a caller's own, what autograd keeps.

Tolerances as in test_route_gpu.py: a weight (k + 16 + |l|) 2^-23 relative, as exponents are differences off by 2^-24
of the larger logit, a gradient (k + 32 + |l|) 2^-23 of its terms' size.
"""

import numpy as np
import pytest
import torch

import spmm_b200 as S

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
INF = float('inf')
STEP = 2.0 ** -23


@pytest.mark.parametrize('renormalize', [True, False])
@pytest.mark.parametrize('centers', [(20.0,), (17.0, -3.0), (-100.0,), (-100.0, -40.0), (-300.0,), (60.0, -95.0)])
@pytest.mark.parametrize('T', [64, 300])
def test_sigmoids_far_from_zero(cuda, renormalize, centers, T):
    """The gradient is held relative to w sigmoid(-l), not to w: 1 - s keeps its bits; weights keep their ratios."""
    torch.manual_seed(21)
    E, k = 24, 5
    l = torch.randn(T, E, device='cuda') * 2 + torch.tensor(centers, device='cuda')[torch.arange(E) % len(centers)]
    bias = torch.randn(E, device='cuda') * 3
    w, r = S.route_topk(l, k, scoring='sigmoid', renormalize=renormalize, bias=bias)
    g = torch.randn(T, k, device='cuda')
    dl = S.route_topk_backward(g, l, r, scoring='sigmoid', renormalize=renormalize)
    at = r.experts.long()
    lj = l.double().gather(1, at)
    share = -torch.logaddexp(torch.zeros_like(lj), -lj)          # log sigmoid
    rest = torch.exp(-torch.logaddexp(torch.zeros_like(lj), lj))  # 1 - sigmoid
    want = torch.softmax(share, 1) if renormalize else torch.exp(share)
    tol = (k + 16 + float(lj.abs().max())) * STEP
    assert ((w.double() - want).abs() <= tol * want + 1e-37).all()
    gd = g.double()
    if renormalize:
        grad = want * (gd - (gd * want).sum(1, keepdim=True)) * rest
        size = 2 * want * gd.abs().amax(1, keepdim=True) * rest
    else:
        grad = want * gd * rest
        size = grad.abs()
    got = dl.double().gather(1, at)
    assert ((got - grad).abs() <= (tol + 16 * STEP) * size + 1e-37).all()
    assert int((dl != 0).sum()) <= T * k


@pytest.mark.parametrize('dtype', [F32, BF, HF])
def test_a_mask_by_the_lowest_value_has_no_share(cuda, dtype):
    l = torch.randn(200, 16, device='cuda').to(dtype)
    l[:, 2:] = torch.finfo(dtype).min
    l[100:] = torch.finfo(dtype).min
    w, r = S.route_topk(l, 4, scoring='sigmoid')
    assert (w[:100, 2:] == 0).all() and ((w[:100].sum(1) - 1).abs() <= 4 * STEP).all() and not w[100:].any()


def test_autograd_allocates_what_the_plain_call_does(cuda):
    l, g = torch.randn(300, 32, device='cuda', requires_grad=True), torch.randn(300, 4, device='cuda')
    w, r = S.route_topk(l, 4)

    def count(call):
        before = torch.cuda.memory_stats()['allocation.all.allocated']
        call()
        return torch.cuda.memory_stats()['allocation.all.allocated'] - before
    plain = count(lambda: S.route_topk_backward(g, l.detach(), r))
    assert count(lambda: torch.autograd.grad(w, l, g)) == plain


def test_gradients_that_never_come(cuda):
    """A later function that gives no gradient at all: none goes on, and nothing is computed."""
    class Stop(torch.autograd.Function):
        @staticmethod
        def forward(ctx, t):
            return t.clone()

        @staticmethod
        def backward(ctx, g):
            return None
    l = torch.randn(40, 8, device='cuda', requires_grad=True)
    x = torch.randn(40, 16, device='cuda').to(BF).requires_grad_()
    w = torch.randn(16, 8, device='cuda').to(BF).requires_grad_()
    y = torch.randn(80, 24, device='cuda').to(BF).requires_grad_()
    weights, r = S.route_topk(l, 2)
    (Stop.apply(weights).sum() + Stop.apply(S.dense_matmul(x, w)).sum()
     + Stop.apply(S.route_combine(y, r, weights.detach())).sum()).backward()
    assert all(t.grad is None for t in (l, x, w, y))


@pytest.mark.parametrize('which', ['slots', 'offsets'])
def test_a_routing_written_again_before_the_backward_pass(cuda, which):
    w, r = S.route_topk(torch.randn(50, 8, device='cuda'), 2)
    y = torch.randn(100, 24, device='cuda').to(BF).requires_grad_()
    out = S.route_combine(y, r, w)
    getattr(r, which).zero_()
    with pytest.raises(RuntimeError, match='inplace'):
        out.sum().backward()


@pytest.mark.parametrize('T, E, k, n, dtype', [(1, 8, 2, 64, BF), (50, 8, 2, 77, HF), (700, 16, 4, 520, BF),
                                               (40, 64, 9, 136, F32), (5000, 8, 3, 24, BF)])
def test_dropped_choices_have_no_gradient(cuda, T, E, k, n, dtype):
    """Slots set to -1 leave rows without a choice: their dy is zero, not what the memory held."""
    torch.manual_seed(T)
    w, r = S.route_topk(torch.randn(T, E, device='cuda'), k)
    slots = torch.where(torch.rand(T, k, device='cuda') < 0.3, -1, r.slots)
    slots[0, 0] = -1
    own = S.Routing(r.experts, slots, r.rows, r.offsets)
    y, d = (torch.randn(s, n, device='cuda').to(dtype) for s in (T * k, T))
    hold = torch.full((T * k, n), float('nan'), device='cuda', dtype=dtype)     # what new_empty may find
    del hold
    dy, dw = S.route_combine_backward(d, y, own, w)
    kept = slots >= 0
    want = torch.zeros(T * k, n, device='cuda', dtype=torch.float64)
    want[slots[kept].long()] = (w.double()[:, :, None] * d.double()[:, None, :])[kept]
    assert ((dy.double() - want).abs() <= (torch.finfo(dtype).eps / 2 + STEP) * want.abs() + 2.0 ** -25).all()
    assert not dw[~kept].any()
    out = S.route_combine(y, own, w)
    part = torch.where(kept[:, :, None], y.double()[slots.clamp(min=0).long()] * w.double()[:, :, None], 0.0)
    lim = (k + 2) * STEP * part.abs().sum(1) + torch.finfo(dtype).eps / 2 * part.sum(1).abs() + 2.0 ** -25
    assert ((out.double() - part.sum(1)).abs() <= lim).all()
