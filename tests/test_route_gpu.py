"""Expert choice, grouping and combination against 64 bits.

Tolerances: a weight is an exponential (or sigmoid) and one division in float32,
with exponents that are differences off by 2^-24 of the larger logit: relative
(E + 16 + |l|) 2^-23.  A gradient adds <g, w> over the chosen ones: (E + 32 +
|l|) 2^-23 of the terms' sizes, and the type's rounding.  Combination: (k + 2)
2^-23 of the terms' sizes and one rounding; its dot products (N + 2) 2^-23.
"""

import numpy as np
import pytest
import torch

import spmm_b200 as S

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
INF = float('inf')
STEP = 2.0 ** -23


def grouping(experts, E):
    flat = experts.reshape(-1)
    live = np.flatnonzero(flat >= 0)
    live = live[np.argsort(flat[live], kind='stable')]
    rows = np.full(flat.size, -1)
    rows[:live.size] = live // experts.shape[1]
    slots = np.full(flat.size, -1)
    slots[live] = np.arange(live.size)
    off = np.concatenate([[0], np.cumsum(np.bincount(flat[live], minlength=E))])
    return slots.reshape(experts.shape), rows, off


def check(logits, top, scoring='softmax', renormalize=True, scale=1.0, bias=None):
    T, E = logits.shape
    weights, r = S.route_topk(logits, top, scoring=scoring, renormalize=renormalize, scale=scale, bias=bias)
    l32 = logits.float().cpu().numpy()
    key = l32 if bias is None else l32 + bias.cpu().numpy()
    key = np.where(np.isnan(key), -np.inf, key)
    order = np.argsort(-key, axis=1, kind='stable')[:, :top]
    ok = np.take_along_axis(key, order, 1) > -np.inf
    experts = np.where(ok, order, -1)
    assert np.array_equal(r.experts.cpu().numpy(), experts)
    slots, rows, off = grouping(experts, E)
    assert np.array_equal(r.slots.cpu().numpy(), slots)
    assert np.array_equal(r.rows.cpu().numpy(), rows)
    assert np.array_equal(r.offsets.cpu().numpy(), off)
    l = np.where(np.isnan(l32), -np.inf, np.minimum(l32, np.finfo(np.float32).max)).astype(np.float64)
    lj = np.take_along_axis(l, order, 1)
    with np.errstate(over='ignore', invalid='ignore', divide='ignore'):
        if scoring == 'softmax':
            base = np.where(ok, lj, -np.inf) if renormalize else l
            m = base.max(1, keepdims=True) if base.size else np.zeros((T, 1))
            m = np.where(np.isfinite(m), m, 0)
            s = np.where(ok, np.exp(lj - m), 0) / np.maximum(np.exp(base - m).sum(1, keepdims=True), 1e-300)
        else:
            s = np.where(ok, 1 / (1 + np.exp(-lj)), 0)
        w = s
        if renormalize:
            tot = s.sum(1, keepdims=True)
            w = s / np.where(tot > 0, tot, 1)
    big = np.abs(np.where(np.isfinite(lj) & ok, lj, 0)).max(initial=0.0)
    big = min(big, 200.0)     # beyond that the exponentials of differences are 0, 1 or equal
    tol = (E + 16 + big) * STEP
    got = weights.cpu().numpy().astype(np.float64)
    assert (np.abs(got - scale * w) <= tol * scale * np.abs(w) + 1e-37).all()
    g = torch.randn(T, top, device='cuda')
    dl = S.route_topk_backward(g, logits, r, scoring=scoring, renormalize=renormalize, scale=scale)
    gd = scale * np.where(ok, g.double().cpu().numpy(), 0)
    dense = np.zeros((T, E))
    size = np.zeros((T, E))
    gabs = np.abs(gd).max(1, keepdims=True, initial=0.0)
    if scoring == 'softmax':
        dot = (gd * w).sum(1, keepdims=True)
        np.put_along_axis(dense, order, np.where(ok, w * (gd - dot), 0), 1)
        np.put_along_axis(size, order, 2 * w * gabs, 1)
        if not renormalize:
            with np.errstate(invalid='ignore'):
                p = np.exp(l - m) / np.maximum(np.exp(l - m).sum(1, keepdims=True), 1e-300)
            rest = np.ones((T, E), bool)
            np.put_along_axis(rest, order, ~ok, 1)
            dense = np.where(rest, -p * dot, dense)
            size = np.where(rest, 2 * p * gabs, size)
    else:
        dot = (gd * w).sum(1, keepdims=True) if renormalize else 0
        np.put_along_axis(dense, order, np.where(ok, w * (gd - dot) * (1 - s), 0), 1)
        np.put_along_axis(size, order, 2 * w * gabs, 1)
    u = torch.finfo(logits.dtype).eps / 2
    err = np.abs(dl.double().cpu().numpy() - dense)
    assert (err <= (E + 32 + big) * STEP * size + u * np.abs(dense) + 2.0 ** -25).all()
    return weights, r


@pytest.mark.parametrize('T, E, k', [(1, 1, 1), (1, 8, 2), (5, 60, 4), (32, 64, 6), (128, 160, 8), (129, 256, 8),
                                     (700, 33, 1), (1000, 512, 3), (300, 1024, 32), (100, 1024, 32), (2500, 128, 8),
                                     (20000, 64, 2)])
@pytest.mark.parametrize('dtype', [F32, BF, HF])
def test_choice_and_grouping(cuda, T, E, k, dtype):
    torch.manual_seed(T + E)
    check((torch.randn(T, E, device='cuda') * 2).to(dtype), k)


@pytest.mark.parametrize('scoring', S.SCORINGS)
@pytest.mark.parametrize('renormalize', [True, False])
@pytest.mark.parametrize('T', [40, 400])
def test_weights_and_gradients(cuda, scoring, renormalize, T):
    torch.manual_seed(1)
    check(torch.randn(T, 96, device='cuda') * 3, 5, scoring, renormalize, 2.5,
          torch.randn(96, device='cuda'))
    check((torch.randn(T, 70, device='cuda') * 3).to(BF), 7, scoring, renormalize)
    check((torch.randn(T, 90, device='cuda') * 3).to(HF), 5, scoring, renormalize, 0.5,
          torch.randn(90, device='cuda') * 2)


@pytest.mark.parametrize('scoring', S.SCORINGS)
@pytest.mark.parametrize('renormalize', [True, False])
@pytest.mark.parametrize('T', [20, 200])
def test_masks(cuda, scoring, renormalize, T):
    """Masked experts, rows with fewer experts than choices, rows without any, the type's lowest value, NaN, ties."""
    torch.manual_seed(2)
    l = torch.randn(T, 40, device='cuda')
    l[0] = -INF
    l[1, 3:] = -INF
    l[2] = float('nan')
    l[3, :38] = float('nan')
    l[4] = torch.finfo(F32).min
    l[5] = 0.0
    l[5, ::2] = -0.0
    l[6, 7:] = l[6, 6]
    l[7, :] = -INF
    l[7, 39] = torch.finfo(F32).min
    l[8, 5] = 300.0
    l[T - 1] = -INF
    check(l, 4, scoring, renormalize)
    check(torch.full((T, 40), -INF, device='cuda'), 4, scoring, renormalize)


def test_plus_infinity_counts_as_the_largest_float(cuda):
    l = torch.zeros(2, 10, device='cuda')
    l[0, 4] = l[0, 7] = INF
    w, r = S.route_topk(l, 3)
    assert r.experts[0].tolist() == [4, 7, 0] and w[0].tolist() == [0.5, 0.5, 0.0]


@pytest.mark.parametrize('T', [0, 1, 3])
def test_few_tokens_and_strides(cuda, T):
    torch.manual_seed(3)
    check(torch.randn(T, 48, device='cuda'), 4)
    check(torch.randn(48, T, device='cuda').t(), 4)
    check(torch.randn(T + 2, 61, device='cuda').to(BF)[1:T + 1, 5:45], 4)


def test_one_expert_takes_all(cuda):
    l = torch.zeros(3000, 64, device='cuda')
    l[:, 63] = 5.0
    check(l, 1)
    check(l, 2)


def combine_ref(y, r, w, res):
    s = r.slots.long()
    ok = (s >= 0)[:, :, None]
    yj = torch.where(ok, y.double()[s.clamp(min=0)], torch.zeros((), dtype=torch.float64, device='cuda'))
    terms = yj * w.double()[:, :, None]
    out, size = terms.sum(1), terms.abs().sum(1)
    if res is not None:
        out, size = out + res.double(), size + res.double().abs()
    return out, size, yj


@pytest.mark.parametrize('T, E, k, n, dtype, masked', [
    (1, 4, 1, 1, BF, 0), (1, 8, 8, 2048, HF, 0), (32, 64, 4, 2048, BF, 3), (33, 6, 3, 77, F32, 2), (300, 16, 5, 520, HF, 0),
    (1000, 8, 2, 1027, BF, 100), (4, 4, 2, 8, BF, 4), (0, 4, 2, 8, BF, 0), (7, 4, 2, 0, BF, 1), (40, 64, 9, 264, F32, 0)])
def test_combine(cuda, T, E, k, n, dtype, masked):
    torch.manual_seed(T + n)
    l = torch.randn(T, E, device='cuda')
    l[T - masked:] = -INF
    w, r = S.route_topk(l, k)
    w = torch.randn_like(w)
    y = torch.randn(T * k, n, device='cuda').to(dtype)
    y[(T - masked) * k:] = float('nan')        # rows of no expert are not read
    res = torch.randn(T, n, device='cuda').to(dtype)
    u = torch.finfo(dtype).eps / 2
    for rr in (None, res, torch.randn(T, n + 3, device='cuda').to(dtype)[:, 3:]):
        want, size, yj = combine_ref(y, r, w, rr)
        out = S.route_combine(y, r, w, rr)
        assert ((out.double() - want).abs() <= (k + 2) * STEP * size + u * want.abs() + 2.0 ** -25).all()
    d = torch.randn(T, n, device='cuda').to(dtype)
    dy, dw = S.route_combine_backward(d, y, r, w)
    terms = yj * d.double()[:, None, :]
    assert ((dw.double() - terms.sum(2)).abs() <= (n + 2) * STEP * terms.abs().sum(2) + 1e-37).all()
    want = torch.zeros(T * k, n, dtype=torch.float64, device='cuda')
    s = r.slots.long()
    want[s[s >= 0]] = (w.double()[:, :, None] * d.double()[:, None, :])[s >= 0]
    assert ((dy.double() - want).abs() <= (u + STEP) * want.abs() + 2.0 ** -25).all()


def test_wrong_slots_stay_inside(cuda):
    w, r = S.route_topk(torch.randn(10, 4, device='cuda'), 2)
    bad = S.Routing(r.experts, r.slots + 1000, r.rows, r.offsets + 1000)
    y = torch.randn(20, 16, device='cuda').to(BF)
    assert not S.route_combine(y, bad, w).any()
    S.route_combine_backward(torch.randn(10, 16, device='cuda').to(BF), y, bad, w)


def test_autograd(cuda):
    torch.manual_seed(9)
    l = torch.randn(50, 16, device='cuda', requires_grad=True)
    w, r = S.route_topk(l, 3, scoring='sigmoid')
    y = torch.randn(150, 40, device='cuda').to(BF).requires_grad_()
    res = torch.randn(50, 40, device='cuda').to(BF).requires_grad_()
    out = S.route_combine(y, r, w, res)
    d = torch.randn(50, 40, device='cuda').to(BF)
    out.backward(d)
    dy, dw = S.route_combine_backward(d, y.detach(), r, w.detach())
    assert torch.equal(y.grad, dy) and torch.equal(res.grad, d)
    assert torch.equal(l.grad, S.route_topk_backward(dw, l.detach(), r, scoring='sigmoid'))


@pytest.mark.parametrize('T', [60, 600])
def test_graph_and_stream(cuda, T):
    torch.manual_seed(T)
    l = torch.randn(T, 64, device='cuda')
    y = torch.randn(T * 4, 128, device='cuda').to(BF)

    def step():
        w, r = S.route_topk(l, 4)
        return w, r.experts, r.slots, r.rows, r.offsets, S.route_combine(y, r, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for seed in range(3):
        torch.manual_seed(seed)
        l.copy_(torch.randn(T, 64, device='cuda'))
        want = step()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
