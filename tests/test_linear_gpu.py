"""Dense and grouped products against 64 bits.

Tolerances, elementwise, with u = eps / 2 of the type (one rounding), S = |x||w|
+ |bias| and E = (K + 8) 2^-23 S for a float32 sum of K products in any order
(each of the K additions off by at most 2^-23 of a partial sum, truncation
included):
  y    1.2 E + 2^-20 |z| + u |y| + 2^-25, as no activation is steeper than 1.13,
       its float32 evaluation is good to a few 2^-23 of |z|, and 2^-25 is half
       the smallest float16
  dz   |dy| (2^-15 + 1.2 E + 2^-20) + u |dz|: the derivative's fixed point, its
       change over E (no second derivative above 1.2), its evaluation, dz's
       rounding; for relu |dy| where |z| <= E
  dx, dw, dbias   the sums of dz's error over |w|, |x|, 1, plus E of their own
       sums and u of the result
"""

import ctypes as C

import pytest
import torch

import spmm_b200 as S
from spmm_b200 import _lib

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
STEP = 2.0 ** -23


def act64(z, name):
    z = z.clone().requires_grad_()
    y = {'none': lambda v: v, 'relu': torch.relu, 'silu': torch.nn.functional.silu,
         'gelu': torch.nn.functional.gelu,
         'gelu_tanh': lambda v: torch.nn.functional.gelu(v, approximate='tanh')}[name](z * 1.0)
    d, = torch.autograd.grad(y.sum(), z)
    return y.detach(), d


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def close(got, want, err, dtype, what):
    lim = err + half_step(dtype) * (want.abs() + err) + 2.0 ** -25
    diff = (got.double() - want).abs()
    bad = ~(diff <= lim)
    assert not bad.any(), f'{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((diff - lim).max()):.3e}'


def group_of(offsets, rows):
    """Group of each row, -1 behind the last one."""
    g = torch.full((rows,), -1, dtype=torch.long)
    o = offsets.tolist()
    for e in range(len(o) - 1):
        g[o[e]:o[e + 1]] = e
    return g


def reference(x, w, gid, src, bias, act, dy):
    """64-bit outputs and error bounds.  w [G,K,N]; row r of the product reads x[src[r]] in group gid[r]."""
    dt, (G, K, N) = x.dtype, w.shape
    R = len(gid)
    dev = x.device
    xd, wd = x.double(), w.double()
    z = torch.zeros(R, N, dtype=torch.float64, device=dev)
    E = torch.zeros_like(z)
    out = {}
    idx = [torch.nonzero(gid == g).flatten().to(dev) for g in range(G)]
    for g in range(G):
        if not len(idx[g]):
            continue
        xs = xd[src[idx[g]]]
        z[idx[g]] = xs @ wd[g]
        E[idx[g]] = xs.abs() @ wd[g].abs()
        if bias is not None:
            z[idx[g]] += bias[g].double()
            E[idx[g]] += bias[g].double().abs()
    E *= (K + 8) * STEP
    y, slope = act64(z, act)
    dead = (gid < 0).to(dev)
    y[dead] = 0
    out['y'] = (y, 1.2 * E + 2.0 ** -20 * z.abs())
    if dy is None:
        return out
    d = dy.double()
    dz = d * slope
    dz[dead] = 0
    ez = torch.zeros_like(dz)
    if act != 'none':
        ez = d.abs() * (2.0 ** -15 + 1.2 * E + 2.0 ** -20)
        if act == 'relu':
            ez = ez + d.abs() * (z.abs() <= E)
        eb = ez.clone()
        ez = ez + half_step(dt) * (dz.abs() + ez) + 2.0 ** -25
    else:
        eb = ez.clone()
    ez[dead] = 0
    eb[dead] = 0
    dx, edx = torch.zeros_like(xd), torch.zeros_like(xd)
    dw, edw = torch.zeros_like(wd), torch.zeros_like(wd)
    db = torch.zeros(G, N, dtype=torch.float64, device=dev)
    edb = torch.zeros_like(db)
    for g in range(G):
        i = idx[g]
        if not len(i):
            continue
        s = src[i]
        dx.index_add_(0, s, dz[i] @ wd[g].t())
        edx.index_add_(0, s, (ez[i] + (N + 16) * STEP * dz[i].abs()) @ wd[g].abs().t())
        dw[g] = xd[s].t() @ dz[i]
        edw[g] = xd[s].abs().t() @ (ez[i] + (len(i) + 8) * STEP * dz[i].abs())
        db[g] = dz[i].sum(0)
        edb[g] = (eb[i] + (len(i) + 8) * STEP * dz[i].abs()).sum(0)
    out.update(dx=(dx, edx), dw=(dw, edw), dbias=(db, edb))
    return out


def check_dense(x, w, bias=None, residual=None, act='none', train=True):
    dt = x.dtype
    dy = torch.randn(x.shape[0], w.shape[1], device='cuda').to(dt) if train else None
    gid = torch.zeros(x.shape[0], dtype=torch.long)
    ref = reference(x, w[None], gid, torch.arange(x.shape[0], device='cuda'), None if bias is None else bias[None],
                    act, dy)
    y, slope = S.dense_matmul(x, w, bias, residual, activation=act, return_slope=True)
    assert S.product_status(y) == 0 and (slope is None) == (act == 'none')
    want, err = ref['y']
    if residual is not None:
        want = want + residual.double()
        err = err + 2 * STEP * want.abs()
    close(y, want, err, dt, 'y')
    assert torch.equal(y, S.dense_matmul(x, w, bias, residual, activation=act))
    if train:
        dx, dw, db = S.dense_matmul_backward(dy, x, w, slope, bias=bias is not None)
        assert S.product_status(dx) == 0
        close(dx, *ref['dx'], dt, 'dx')
        close(dw, ref['dw'][0][0], ref['dw'][1][0], dt, 'dw')
        if bias is not None:
            close(db, ref['dbias'][0][0], ref['dbias'][1][0], dt, 'dbias')


def normal(*shape, dtype=BF, scale=1.0):
    return (torch.randn(*shape, device='cuda') * scale).to(dtype)


@pytest.mark.parametrize('act', S.ACTIVATIONS)
@pytest.mark.parametrize('t, k, n, dtype', [
    (1, 1, 1, BF), (3, 17, 9, HF), (16, 64, 128, BF), (130, 72, 264, HF), (65, 200, 100, BF), (257, 321, 513, BF),
    (300, 1024, 640, HF)])
def test_dense(cuda, t, k, n, dtype, act):
    torch.manual_seed(t + k + n)
    check_dense(normal(t, k, dtype=dtype), normal(k, n, dtype=dtype, scale=k ** -0.5), normal(n, dtype=dtype),
                normal(t, n, dtype=dtype), act)


@pytest.mark.parametrize('t, k, n', [(1, 4096, 4096), (7, 2048, 512), (33, 1000, 2504), (64, 8192, 136),
                                     (1025, 640, 1288), (2048, 64, 64), (4100, 128, 72)])
@pytest.mark.parametrize('w_t', [False, True])
def test_dense_shapes(cuda, t, k, n, w_t):
    torch.manual_seed(t * 3 + n)
    w = normal(n, k, scale=k ** -0.5).t() if w_t else normal(k, n, scale=k ** -0.5)
    check_dense(normal(t, k), w, act='silu')


def test_dense_strides_and_alignment(cuda):
    torch.manual_seed(5)
    big = normal(70, 300)
    x = big[3:60, 1:202]                       # odd base and row stride
    wbig = normal(250, 333, scale=0.1)
    for w in (wbig[5:206, 7:140], wbig.t()[5:206, 7:140], wbig[:201, :133].t().contiguous().t(),
              normal(402, 133, scale=0.1)[::2]):
        check_dense(x, w, normal(266)[::2], normal(57, 300)[:, 5:138], act='gelu')
    check_dense(normal(201, 57).t(), wbig[:201, :133])                       # transposed x
    check_dense(x, normal(1, 133, scale=0.1).expand(201, 133), act='silu')   # broadcast w
    r = normal(1, 133).expand(57, 133)                                       # broadcast residual
    check_dense(x, wbig[:201, :133], None, r, train=False)


@pytest.mark.parametrize('t, k, n', [(0, 5, 7), (5, 0, 7), (5, 7, 0), (0, 0, 0), (130, 0, 300)])
def test_dense_empty(cuda, t, k, n):
    check_dense(normal(t, k), normal(k, n), normal(n), normal(t, n), 'gelu')


def test_dense_leading_dimensions(cuda):
    x, w, r = normal(2, 3, 5, 24), normal(24, 16), normal(2, 3, 5, 16)
    y = S.dense_matmul(x, w, None, r, activation='relu')
    assert y.shape == r.shape and S.product_status(y) == 0
    assert torch.equal(y.reshape(30, 16), S.dense_matmul(x.reshape(30, 24), w, None, r.reshape(30, 16),
                                                         activation='relu'))
    assert S.dense_matmul(x[0, 0, 0], w).shape == (16,)


@pytest.mark.parametrize('act', S.ACTIVATIONS)
def test_infinities_stay_in_their_rows(cuda, act):
    x, w = normal(40, 96), normal(96, 80)
    base = S.dense_matmul(x, w, activation=act)
    x2 = x.clone()
    x2[3, 5], x2[17, 0], x2[39, 95] = float('nan'), float('inf'), float('-inf')
    y = S.dense_matmul(x2, w, activation=act)
    keep = torch.ones(40, dtype=torch.bool, device='cuda')
    keep[[3, 17, 39]] = False
    assert torch.equal(y[keep], base[keep])
    want, _ = act64((x2.double() @ w.double())[~keep], act)
    got = y[~keep].double()
    assert torch.equal(torch.isnan(got[0]), torch.isnan(want[0])) and torch.isnan(got[0]).all()
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])


def test_large_values_saturate_like_a_rounding(cuda):
    x = torch.full((4, 64), 200.0, device='cuda', dtype=HF)
    w = torch.full((64, 8), 200.0, device='cuda', dtype=HF)
    assert torch.isinf(S.dense_matmul(x, w)).all()           # 2.56e6 is over float16's range
    assert torch.equal(S.dense_matmul(x, -w, activation='silu'), torch.zeros(4, 8, device='cuda', dtype=HF))


CASES = [   # lengths of the groups, rows behind the last one, k, n
    ([5], 0, 24, 40), ([0, 0, 0], 0, 16, 16), ([0, 7, 0, 1, 0], 3, 33, 65), ([1] * 40, 0, 256, 136),
    ([300, 0, 1, 65, 64, 129], 11, 128, 264), ([17, 250, 3], 130, 72, 520), ([16, 32, 48, 15, 31], 0, 512, 192),
    ([513, 2], 1, 320, 328)]


@pytest.mark.parametrize('lens, tail, k, n', CASES)
@pytest.mark.parametrize('dtype, act, w_t', [(BF, 'none', False), (HF, 'silu', True), (BF, 'gelu', True),
                                             (BF, 'relu', False)])
def test_grouped(cuda, lens, tail, k, n, dtype, act, w_t):
    torch.manual_seed(len(lens) + k)
    G, R = len(lens), sum(lens) + tail
    offsets = torch.tensor([0] + lens).cumsum(0).int()
    x = normal(R, k, dtype=dtype)
    w = normal(G, n, k, dtype=dtype, scale=k ** -0.5).transpose(1, 2) if w_t else normal(G, k, n, dtype=dtype,
                                                                                        scale=k ** -0.5)
    bias, dy = normal(G, n, dtype=dtype), normal(R, n, dtype=dtype)
    x[R - tail:] = float('nan')              # rows of no group touch nothing
    dy[R - tail:] = float('inf')
    xr, dr = x.clone(), dy.clone()
    xr[R - tail:], dr[R - tail:] = 0, 0
    ref = reference(xr, w, group_of(offsets, R), torch.arange(R, device='cuda'), bias, act, dr)
    go = offsets.cuda()
    y, slope = S.grouped_matmul(x, w, go, bias, activation=act, return_slope=True)
    close(y, *ref['y'], dtype, 'y')
    dx, dw, db = S.grouped_matmul_backward(dy, x, w, go, slope, bias=True)
    assert S.product_status(y) == 0 and S.product_status(dw) == 0
    for name, got in (('dx', dx), ('dw', dw), ('dbias', db)):
        close(got, *ref[name], dtype, name)
    assert dw.stride() == w.stride()
    again = S.grouped_matmul_backward(dy, x, w, go, slope, bias=True)
    assert all(torch.equal(a, b) for a, b in zip((dx, dw, db), again))


@pytest.mark.parametrize('tokens, experts, top, k, n, masked', [
    (1, 4, 1, 64, 64, 0), (3, 8, 8, 40, 24, 1), (50, 16, 3, 136, 72, 5), (200, 64, 6, 256, 128, 0),
    (600, 5, 2, 65, 130, 20), (2500, 9, 4, 328, 392, 77), (900, 64, 8, 192, 264, 0),
    (10, 64, 6, 136, 72, 2)])
@pytest.mark.parametrize('w_t', [False, True])
def test_grouped_gather(cuda, tokens, experts, top, k, n, masked, w_t):
    torch.manual_seed(tokens)
    logits = torch.randn(tokens, experts, device='cuda')
    logits[tokens - masked:] = float('-inf')
    weights, r = S.route_topk(logits, top)
    x, w = normal(tokens, k), normal(experts, k, n, scale=k ** -0.5)
    if w_t:
        w = w.transpose(1, 2).contiguous().transpose(1, 2)
    dy = normal(tokens * top, n)
    gid = group_of(r.offsets.cpu(), tokens * top)
    src = r.rows.long().clamp(min=0)
    ref = reference(x, w, gid, src, None, 'silu', dy)
    y, slope = S.grouped_matmul(x, w, r, activation='silu', gather=True, return_slope=True)
    close(y, *ref['y'], BF, 'y')
    dx, dw, _ = S.grouped_matmul_backward(dy, x, w, r, slope, gather=True)
    close(dx, *ref['dx'], BF, 'dx')
    close(dw, *ref['dw'], BF, 'dw')
    # the same as with the rows laid out by the caller
    assert torch.equal(y[gid >= 0], S.grouped_matmul(x[src], w, r, activation='silu')[gid >= 0])


@pytest.mark.parametrize('t, k, n', [(3000, 256, 6200), (700, 2048, 4096), (5000, 520, 1500)])
def test_many_tiles(cuda, t, k, n):
    """More tiles than SMs: several per CTA, both accumulators in use."""
    torch.manual_seed(t)
    check_dense(normal(t, k), normal(k, n, scale=k ** -0.5), normal(n), normal(t, n), 'gelu_tanh')


@pytest.mark.parametrize('t, k, n', [(70001, 64, 72), (3, 72, 70000), (5, 70000, 8)])
def test_long_dimensions(cuda, t, k, n):
    torch.manual_seed(t)
    check_dense(normal(t, k), normal(k, n, scale=k ** -0.5), normal(n), None, 'silu')


@pytest.mark.parametrize('t, k, n', [(70000, 32768, 16), (70000, 16, 32768)])
def test_offsets_past_32_bits(cuda, t, k, n):
    """x, or y and the slopes, of more than 2**31 values: the last rows against the same rows alone."""
    torch.manual_seed(k)
    x, w = torch.empty(t, k, device='cuda', dtype=BF).normal_(), normal(k, n, scale=k ** -0.5)
    y, slope = S.dense_matmul(x, w, activation='silu', return_slope=True)
    z = x[-70:].double() @ w.double()
    want, d = act64(z, 'silu')
    E = (k + 8) * STEP * (x[-70:].double().abs() @ w.double().abs())
    close(y[-70:], want, 1.2 * E + 2.0 ** -20 * z.abs(), BF, 'y')
    assert ((slope[-70:].double() / 16384 - d).abs() <= 2.0 ** -15 + 1.2 * E + 2.0 ** -20).all()
    dx, dw, _ = S.dense_matmul_backward(y, x, w, None)
    tail = S.dense_matmul_backward(y[-70:], x[-70:], w, None)[0]
    bound = (n + 16) * STEP * (y[-70:].double().abs() @ w.double().abs().t())
    close(dx[-70:], y[-70:].double() @ w.double().t(), bound, BF, 'dx')
    close(tail, y[-70:].double() @ w.double().t(), bound, BF, 'dx of the tail')
    assert torch.isfinite(dw).all()


def test_one_group_takes_all_rows(cuda):
    """The kernel for a handful of rows is chosen by their average; one group may still have them all."""
    torch.manual_seed(8)
    x, w = normal(31, 256), normal(32, 256, 136, scale=1 / 16)
    for g in (0, 17, 31):
        offsets = torch.zeros(33, dtype=torch.int32)
        offsets[g + 1:] = 29
        y = S.grouped_matmul(x, w, offsets.cuda(), activation='gelu')
        ref = reference(x, w, group_of(offsets, 31), torch.arange(31, device='cuda'), None, 'gelu', None)
        close(y, *ref['y'], BF, 'y')


def test_many_ragged_groups(cuda):
    torch.manual_seed(11)
    G, k, n = 200, 192, 328
    lens = [int(v) for v in torch.randint(0, 90, (G,))]
    lens[17], lens[100] = 900, 0
    offsets = torch.tensor([0] + lens).cumsum(0).int()
    R = sum(lens) + 40
    x, w, b, dy = normal(R, k), normal(G, k, n, scale=k ** -0.5), normal(G, n), normal(R, n)
    ref = reference(x, w, group_of(offsets, R), torch.arange(R, device='cuda'), b, 'silu', dy)
    go = offsets.cuda()
    y, slope = S.grouped_matmul(x, w, go, b, activation='silu', return_slope=True)
    close(y, *ref['y'], BF, 'y')
    for name, got in zip(('dx', 'dw', 'dbias'), S.grouped_matmul_backward(dy, x, w, go, slope, bias=True)):
        close(got, *ref[name], BF, name)


def test_expired_wait_is_reported(cuda):
    """A wait that nothing ends runs out after wait_us; the call's status says so and the next call is unharmed."""
    x, w = normal(300, 256), normal(256, 512)
    y = torch.zeros(300, 512, device='cuda', dtype=BF)
    status = torch.full((1,), 7, dtype=torch.int32, device='cuda')
    a = _lib.Linear()
    a.version, a.dtype, a.rows, a.x_rows, a.k, a.n, a.groups = 1, _lib.DENSE_BF16, 300, 300, 256, 512, 1
    a.x, a.x_ld, a.w, a.w_k, a.w_n, a.y, a.y_ld = x.data_ptr(), 256, w.data_ptr(), 512, 1, y.data_ptr(), 512
    a.status, a.wait_us, a.flags = status.data_ptr(), 2000, _lib.SPMM_CFG_EXPIRE_FIRST_WAIT
    ws = torch.empty(_lib.lib().spmm_linear_forward_workspace_size(C.byref(a)) + 256, device='cuda', dtype=torch.uint8)
    a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    stream = torch.cuda.current_stream().cuda_stream
    assert _lib.lib().spmm_linear_forward(C.byref(a), stream) == 0
    torch.cuda.synchronize()
    assert int(status) == _lib.SPMM_ETIMEOUT
    a.flags = a.wait_us = 0
    assert _lib.lib().spmm_linear_forward(C.byref(a), stream) == 0
    torch.cuda.synchronize()
    assert int(status) == 0 and torch.equal(y, S.dense_matmul(x, w))


def test_wrong_offsets_stay_inside(cuda):
    x, w = normal(50, 64), normal(4, 64, 64)
    for o in ([0, 60, 70, 80, 90], [0, 30, 10, 40, 50], [-5, 10, 20, 30, 40], [7, 7, 7, 7, 7]):
        o = torch.tensor(o, dtype=torch.int32, device='cuda')
        y, slope = S.grouped_matmul(x, w, o, activation='relu', return_slope=True)
        S.grouped_matmul_backward(x, x, w, o, slope, bias=True)
        assert S.product_status(y) == 0


def test_gradients_against_differences(cuda):
    """The formula's gradients: float64 differences of float64 products bound the kernel's float16 gradients."""
    torch.manual_seed(2)
    x, w, b, dy = (normal(6, 8, dtype=HF), normal(8, 5, dtype=HF, scale=0.3), normal(5, dtype=HF),
                   normal(6, 5, dtype=HF))
    for act in ('silu', 'gelu', 'gelu_tanh'):
        _, slope = S.dense_matmul(x, w, b, activation=act, return_slope=True)
        grads = S.dense_matmul_backward(dy, x, w, slope, bias=True)
        args = [x.double(), w.double(), b.double()]

        def f(a):
            return (act64(a[0] @ a[1] + a[2], act)[0] * dy.double()).sum()
        for i, g in enumerate(grads):
            h = 1e-5
            for at in range(args[i].numel()):
                hi, lo = [a.clone() for a in args], [a.clone() for a in args]
                hi[i].view(-1)[at] += h
                lo[i].view(-1)[at] -= h
                diff = float((f(hi) - f(lo)) / (2 * h))
                # sums of at most 8 terms of size |dy w| < 16: 8 * 16 * (2^-15 + 2^-11) for dz, u of the result
                assert abs(float(g.reshape(-1)[at]) - diff) <= 128 * (2.0 ** -15 + 2.0 ** -11) + 2.0 ** -11 * abs(diff)


def test_autograd_matches_the_plain_calls(cuda):
    torch.manual_seed(3)
    x, w, b, r = normal(30, 48), normal(48, 56), normal(56), normal(30, 56)
    leaves = [t.clone().requires_grad_() for t in (x, w, b, r)]
    dy = normal(30, 56)
    y = S.dense_matmul(*leaves, activation='gelu')
    assert S.product_status(y) == 0
    y.backward(dy)
    y2, slope = S.dense_matmul(x, w, b, r, activation='gelu', return_slope=True)
    want = S.dense_matmul_backward(dy, x, w, slope, bias=True) + (dy,)
    assert torch.equal(y, y2) and all(torch.equal(a.grad, g) for a, g in zip(leaves, want))
    xl = x.clone().requires_grad_()           # only some inputs ask for a gradient
    S.dense_matmul(xl, w, b).backward(dy)
    assert torch.equal(xl.grad, S.dense_matmul_backward(dy, x, w)[0])
    e = normal(1, 56).requires_grad_()        # an expanded residual sums its gradient
    S.dense_matmul(x, w, None, e.expand(30, 56)).sum().backward()
    assert torch.equal(e.grad, torch.full((1, 56), 30.0, device='cuda', dtype=BF))
    with torch.no_grad():
        assert not S.dense_matmul(*leaves).requires_grad


def test_single_gradients(cuda):
    """One input at a time asks for a gradient, dense and grouped, with and without an activation."""
    torch.manual_seed(6)
    x, w, b, r, dy = normal(70, 40), normal(40, 24), normal(24), normal(70, 24), normal(70, 24)
    offsets = torch.tensor([0, 30, 30, 70], dtype=torch.int32, device='cuda')
    wg, bg = normal(3, 40, 24), normal(3, 24)
    for act in ('none', 'silu'):
        _, slope = S.dense_matmul(x, w, b, r, activation=act, return_slope=True)
        want = S.dense_matmul_backward(dy, x, w, slope, bias=True) + (dy,)
        for i in range(4):
            args = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, w, b, r))]
            g, = torch.autograd.grad(S.dense_matmul(*args, activation=act), args[i], dy)
            assert torch.equal(g, want[i]), (act, i)
        _, slope = S.grouped_matmul(x, wg, offsets, bg, activation=act, return_slope=True)
        want = S.grouped_matmul_backward(dy, x, wg, offsets, slope, bias=True)
        for i in range(3):
            args = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, wg, bg))]
            y = S.grouped_matmul(args[0], args[1], offsets, args[2], activation=act)
            g, = torch.autograd.grad(y, args[i], dy)
            assert torch.equal(g, want[i]), (act, i)


@pytest.mark.parametrize('tokens, masked', [(0, 0), (9, 9)])
def test_no_rows_at_all(cuda, tokens, masked):
    """No tokens, or none that any expert takes: zeros everywhere, the experts' gradients among them."""
    logits = torch.randn(tokens, 6, device='cuda')
    logits[tokens - masked:] = float('-inf')
    weights, r = S.route_topk(logits, 2)
    x, w, b = normal(tokens, 32), normal(6, 32, 24), normal(6, 24)
    y, slope = S.grouped_matmul(x, w, r, b, activation='gelu', gather=True, return_slope=True)
    assert y.shape == (2 * tokens, 24) and not y.any() and S.product_status(y) == 0
    dx, dw, db = S.grouped_matmul_backward(normal(2 * tokens, 24), x, w, r, slope, gather=True, bias=True)
    assert dx.shape == x.shape and not dx.any() and not dw.any() and not db.any()
    out = S.route_combine(y, r, weights)
    assert out.shape == (tokens, 24) and not out.any()


def test_calls_from_two_threads(cuda):
    import threading
    torch.manual_seed(12)
    x, w = normal(300, 512), normal(512, 640)
    want = S.dense_matmul(x, w, activation='silu')
    bad = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                y = S.dense_matmul(x, w, activation='silu')
                torch.cuda.current_stream().synchronize()
                if not torch.equal(y, want):
                    bad.append(1)
    torch.cuda.synchronize()
    threads = [threading.Thread(target=work) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_streams_and_graphs(cuda):
    torch.manual_seed(4)
    lens = [70, 0, 3, 129]
    offsets = torch.tensor([0] + lens).cumsum(0).int().cuda()
    x, w, b, dy = normal(202, 136), normal(4, 136, 72), normal(4, 72), normal(202, 72)

    def step(x, dy):
        y, slope = S.grouped_matmul(x, w, offsets, b, activation='silu', return_slope=True)
        return (y,) + S.grouped_matmul_backward(dy, x, w, offsets, slope, bias=True)

    want = step(x, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x, dy)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(want, got))
    # two graphs, replayed in turn and overlapping, with new inputs
    bufs = [(x.clone(), dy.clone()) for _ in range(2)]
    outs, graphs = [], []
    with torch.cuda.stream(side):
        for bx, bd in bufs:
            step(bx, bd)
    torch.cuda.synchronize()
    for bx, bd in bufs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(bx, bd))
        graphs.append(g)
    x2, dy2 = normal(202, 136), normal(202, 72)
    bufs[1][0].copy_(x2)
    bufs[1][1].copy_(dy2)
    want2 = step(x2, dy2)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graphs[0].replay()
    graphs[1].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(want, outs[0]))
    assert all(torch.equal(a, c) for a, c in zip(want2, outs[1]))
    graphs[0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(want, outs[0]))


def test_capture_while_an_eager_graph_lives(cuda):
    """The plain calls build no autograd graph: captured with leaves that an eager graph still holds."""
    torch.manual_seed(13)
    leaves = [t.requires_grad_() for t in (normal(64, 48), normal(48, 80), normal(80))]
    eager = S.dense_matmul(*leaves, activation='gelu')
    dy = normal(64, 80)

    def step():
        y, slope = S.dense_matmul(*leaves, activation='gelu', return_slope=True)
        assert not y.requires_grad
        return (y,) + S.dense_matmul_backward(dy, leaves[0], leaves[1], slope, bias=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    g.replay()
    torch.cuda.synchronize()
    eager.backward(dy)
    assert torch.equal(got[0], eager.detach())
    assert all(torch.equal(a, t.grad) for a, t in zip(got[1:], leaves))


def test_expert_layer(cuda):
    """Router, both expert products, the way back and a shared dense part together, with gradients, against
    float64 autograd over the same choices.  Bounds: relative to the largest element of each result, the chain's
    four roundings forward (hidden, expert output, shared, sum) and about six backward, each u = 2^-8 of a sum
    whose terms are at most a few times larger than it: 6 * 2^-8 * 4 < 0.1."""
    torch.manual_seed(7)
    T, E, k, D, H = 90, 12, 3, 128, 192
    x, wr = normal(T, D, scale=0.5), normal(D, E, scale=D ** -0.5)
    w1, w2 = normal(E, D, H, scale=D ** -0.5), normal(E, H, D, scale=H ** -0.5)
    ws, bs = normal(D, D, scale=D ** -0.5), normal(D)
    leaves = [t.clone().requires_grad_() for t in (x, wr, w1, w2, ws, bs)]

    def layer(x, wr, w1, w2, ws, bs):
        weights, r = S.route_topk(S.dense_matmul(x, wr), k)
        h = S.grouped_matmul(x, w1, r, activation='silu', gather=True)
        shared = S.dense_matmul(x, ws, bs, x, activation='gelu')
        return S.route_combine(S.grouped_matmul(h, w2, r), r, weights, shared), r

    out, r = layer(*leaves)
    dy = normal(T, D)
    out.backward(dy)
    d = [t.double().requires_grad_() for t in (x, wr, w1, w2, ws, bs)]
    p = torch.softmax((d[0] @ d[1]), 1).gather(1, r.experts.long())
    p = p / p.sum(1, keepdim=True)
    e = r.experts.long()
    ref = torch.nn.functional.gelu(d[0] @ d[4] + d[5]) + d[0]
    for j in range(k):
        h = torch.nn.functional.silu(torch.einsum('td,tdh->th', d[0], d[2][e[:, j]]))
        ref = ref + p[:, j, None] * torch.einsum('th,thd->td', h, d[3][e[:, j]])
    ref.backward(dy.double())
    assert (out.double() - ref).abs().max() <= 0.1 * ref.abs().max()
    for a, b in zip(leaves, d):
        assert (a.grad.double() - b.grad).norm() <= 0.1 * b.grad.norm()
