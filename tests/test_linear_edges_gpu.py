"""Dense and grouped products at the edges of what their entries accept: wrong tables, scratch that ends where its
size says, combinations that only the C entries take, far sizes, and what autograd keeps.

Tolerances are those of test_linear_gpu.py: u = eps / 2 of the type for the one rounding of a result, and
(K + 8) 2^-23 |x||w| for a float32 sum of K products.
"""

import ctypes as C

import pytest
import torch

import spmm_b200 as S
from spmm_b200 import _lib

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
STEP = 2.0 ** -23


def normal(*shape, dtype=BF, scale=1.0):
    return (torch.randn(*shape, device='cuda') * scale).to(dtype)


def int32(*values):
    return torch.tensor(values, dtype=torch.int32, device='cuda')


def linear(rows, k, n, groups=1, dtype=_lib.DENSE_BF16, **kw):
    """A filled spmm_linear; tensors are given as tensors."""
    a = _lib.Linear()
    a.version, a.dtype, a.rows, a.x_rows, a.k, a.n, a.groups = 1, dtype, rows, rows, k, n, groups
    a.x_ld = a.dx_ld = k
    a.w_k = a.y_ld = a.dy_ld = a.residual_ld = a.bias_g = a.dbias_g = a.dw_k = n
    a.w_n = a.dw_n = 1
    a.w_g = a.dw_g = k * n
    for name, v in kw.items():
        setattr(a, name, v.data_ptr() if isinstance(v, torch.Tensor) else v)
    a.keep = kw            # the tensors live as long as the struct
    return a


def run(name, a, before=0, after=256):
    """Runs a C entry with exactly its workspace, in the middle of a buffer of NaNs; returns the buffer and where in
    it the workspace lay."""
    L = _lib.lib()
    need = getattr(L, name + '_workspace_size')(C.byref(a))
    buf = torch.full((before + need + after,), 0xFF, dtype=torch.uint8, device='cuda')
    buf[before:before + need] = 0
    a.workspace, a.workspace_bytes = buf.data_ptr() + before, need
    assert getattr(L, name)(C.byref(a), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    return buf, before, before + need


def test_decreasing_offsets_read_nothing_behind_the_workspace(cuda):
    """offsets 0, R, 0, R, ...: every second group has all rows, far more tiles in all than rows alone would have."""
    G, R, n = 300, 6400, 8
    offsets = int32(*([0, R] * (G // 2 + 1))[:G + 1])
    dy, dbias = normal(R, n), torch.empty(G, n, device='cuda', dtype=BF)
    a = linear(R, 8, n, G, offsets=offsets, dy=dy, dbias=dbias)
    # 15,000 tiles of 8 float32 before the last group: the guards reach further than that either way
    buf, lo, hi = run('spmm_linear_backward', a, 1 << 20, 1 << 20)
    assert torch.isfinite(dbias).all() and not dbias[1::2].any()
    assert (buf[:lo] == 0xFF).all() and (buf[hi:] == 0xFF).all()


def test_bias_gradients_of_groups_that_end_within_a_tile(cuda):
    """Lengths around the tile of 64 rows, empty groups between them: each group's sum is its own."""
    torch.manual_seed(1)
    lens = [64, 0, 1, 63, 65, 0, 0, 128, 127, 129, 1, 1, 62, 64]
    offsets = int32(0, *torch.tensor(lens).cumsum(0).tolist())
    R, n = sum(lens) + 70, 136
    x, w, dy = normal(R, 8), normal(len(lens), 8, n), normal(R, n)
    db = S.grouped_matmul_backward(dy, x, w, offsets, bias=True)[2].double()
    at = 0
    for g, m in enumerate(lens):
        rows = dy[at:at + m].double()
        want, size = rows.sum(0), rows.abs().sum(0)
        assert ((db[g] - want).abs() <= 2.0 ** -8 * want.abs() + (m + 8) * STEP * size * 1.01 + 2.0 ** -25).all(), g
        at += m


@pytest.mark.parametrize('table', [[0, 300, 100, 400, 250, 500], [0, 520, 0, 520, 0, 520], [400, 300, 200, 100, 0, 50],
                                   [-7, 200, 900, 100, 1000, 300]])
@pytest.mark.parametrize('n', [72, 640])
def test_decreasing_offsets_count_as_their_running_maximum(cuda, table, n):
    """On the tensor cores no two groups own the same row, whatever the table says; the first one starts at 0."""
    torch.manual_seed(2)
    R, k = 520, 136
    x, w, dy = normal(R, k), normal(5, k, n, scale=k ** -0.5), normal(R, n)
    wrong = int32(*table)
    right = int32(0, *table[1:]).clamp(0, R).cummax(0).values.int()
    assert torch.equal(S.grouped_matmul(x, w, wrong), S.grouped_matmul(x, w, right))
    got, want = S.grouped_matmul_backward(dy, x, w, wrong), S.grouped_matmul_backward(dy, x, w, right)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert S.product_status(got[0]) == 0


@pytest.mark.parametrize('rows, k, n', [(1, 256, 136), (64, 8192, 136), (700, 64, 264), (3, 17, 9), (5, 0, 24)])
@pytest.mark.parametrize('act', [0, 1])
def test_slope_of_every_kernel(cuda, rows, k, n, act):
    """A slope that is asked for is written whichever kernel the sizes choose, also where there is no activation."""
    torch.manual_seed(3)
    x, w = normal(rows, k), normal(k, n, scale=max(k, 1) ** -0.5)
    y = torch.empty(rows, n, device='cuda', dtype=BF)
    slope = torch.full((rows, n), 77, device='cuda', dtype=torch.int16)
    run('spmm_linear_forward', linear(rows, k, n, x=x, w=w, y=y, slope=slope, activation=act))
    z = x.double() @ w.double()
    sure = z.abs() > (k + 8) * STEP * (x.double().abs() @ w.double().abs())
    want = torch.full_like(slope, 16384) if act == 0 else torch.where(z > 0, 16384, 0).short()
    assert torch.equal(slope[sure], want[sure]) if act else torch.equal(slope, want)


def test_slope_of_rows_behind_the_last_group(cuda):
    for R, end in ((300, 190), (40, 9)):
        x, w = normal(R, 64), normal(2, 64, 72)
        y = torch.empty(R, 72, device='cuda', dtype=BF)
        slope = torch.full((R, 72), 77, device='cuda', dtype=torch.int16)
        run('spmm_linear_forward', linear(R, 64, 72, 2, x=x, w=w, y=y, slope=slope, offsets=int32(0, 5, end)))
        assert (slope[:end] == 16384).all() and not slope[end:].any() and not y[end:].any()


def points(lo, hi):
    """z = x + bias exactly: x in steps of 2^-10 (float16 has them up to 2, then 2^-9), bias in steps of 2^-16."""
    x = torch.arange(int(lo * 1024), int(hi * 1024) + 1, device='cuda').double() / 1024
    x = x.to(HF)[:, None]
    bias = (torch.arange(64, device='cuda').double() / 65536).to(HF)
    return x, bias, x.double() + bias.double()


def test_derivative_of_tanh_gelu(cuda):
    """The derivative's fixed point is half a unit off, 2^-15, and its float32 evaluation, with s the sigmoid of u =
    1.6 z (1 + 0.045 z^2), q = 1.6 + 0.21 z^2 and d = s + z s (1 - s) q: u |u| 5 2^-24 off, the hardware's exponential
    and reciprocal 2^-22 and 2^-23 of theirs, so s at most 1.3e-6 s; d changes by 1 + z q (1 - 2 s) times that and
    four roundings of its second term: below 3e-7 for all z in [-2.2, -1]."""
    x, bias, z = points(-2.2, -1.0)
    w = torch.ones(1, 64, device='cuda', dtype=HF)
    _, slope = S.dense_matmul(x, w, bias, activation='gelu_tanh', return_slope=True)
    c = (2 / torch.pi) ** 0.5
    t = torch.tanh(c * (z + 0.044715 * z ** 3))
    want = 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    assert ((slope.double() / 16384 - want).abs() <= 2.0 ** -15 + 3e-7).all()


def test_gelu_keeps_its_bits_far_from_zero(cuda):
    """z erfc(-z / sqrt 2) / 2 for z in [-10, -1]: the exponent z^2 / 2 is two roundings and a constant off, 2.5 2^-24
    of it, so 7.5e-6 at z = -10; the exponential 2^-22, the polynomial 4e-7, its argument 2^-23, three products 2^-24:
    below 1.1e-5 before the rounding to bfloat16."""
    x = torch.arange(-10 * 32, -31, device='cuda').double().div(32).to(BF)[:, None]
    bias = (torch.arange(64, device='cuda').double() / 65536).to(BF)
    z = x.double() + bias.double()
    y = S.dense_matmul(x, torch.ones(1, 64, device='cuda', dtype=BF), bias, activation='gelu')
    want = 0.5 * z * torch.special.erfc(-z / 2 ** 0.5)
    assert ((y.double() - want).abs() <= (2.0 ** -8 + 1.1e-5 * (1 + 2.0 ** -8)) * want.abs()).all()


def allocations(call):
    before = torch.cuda.memory_stats()['allocation.all.allocated']
    call()
    return torch.cuda.memory_stats()['allocation.all.allocated'] - before


def test_autograd_allocates_what_the_plain_call_does(cuda):
    x, w, b, dy = normal(64, 48), normal(48, 80), normal(80), normal(64, 80)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    _, slope = S.dense_matmul(x, w, b, activation='silu', return_slope=True)
    plain = allocations(lambda: S.dense_matmul_backward(dy, x, w, slope, bias=True))
    y = S.dense_matmul(*leaves, activation='silu')
    # one less: the forward pass's status word speaks for the backward pass too
    assert allocations(lambda: torch.autograd.grad(y, leaves, dy)) == plain - 1


@pytest.mark.parametrize('which', ['offsets', 'rows', 'slots'])
def test_a_grouping_written_again_before_the_backward_pass(cuda, which):
    _, r = S.route_topk(torch.randn(50, 8, device='cuda'), 2)
    x, w = normal(50, 40).requires_grad_(), normal(8, 40, 24).requires_grad_()
    y = S.grouped_matmul(x, w, r, gather=True)
    getattr(r, which).zero_()
    with pytest.raises(RuntimeError, match='inplace'):
        y.sum().backward()
    offsets = int32(0, 20, 50)
    y = S.grouped_matmul(x, w[:2], offsets)
    offsets += 1
    with pytest.raises(RuntimeError, match='inplace'):
        y.sum().backward()


@pytest.mark.parametrize('rows, grouped', [(2, False), (70, False), (70, True)])
def test_gradients_of_very_wide_results(cuda, rows, grouped):
    """More columns than 65,535 blocks of 256.  dy is 0 but in a first and a last strip, so that the sums over n have
    600 terms; N in the bound counts those."""
    torch.manual_seed(9)
    k, n = 8, 65535 * 256 + 320
    at = torch.cat((torch.arange(300), torch.arange(n - 300, n))).cuda()
    x, w = normal(rows, k), normal(k, n, scale=k ** -0.5)
    dy = torch.zeros(rows, n, device='cuda', dtype=BF)
    dy[:, at] = normal(rows, 600)
    y, slope = (S.grouped_matmul(x, w[None], int32(0, rows), activation='silu', return_slope=True) if grouped else
                S.dense_matmul(x, w, activation='silu', return_slope=True))
    dx, dw, db = (S.grouped_matmul_backward(dy, x, w[None], int32(0, rows), slope, bias=True) if grouped else
                  S.dense_matmul_backward(dy, x, w, slope, bias=True))
    dw, db = dw.reshape(k, n), db.reshape(n)
    z = x.double() @ w[:, at].double()
    s = torch.sigmoid(z)
    d = s * (1 + z * (1 - s))
    E = (k + 8) * STEP * (x.double().abs() @ w[:, at].double().abs())
    dz = dy[:, at].double() * d
    eb = dy[:, at].double().abs() * (2.0 ** -15 + 1.2 * E + 2.0 ** -20)
    ez = eb + 2.0 ** -8 * (dz.abs() + eb)

    def close(got, want, err):
        assert ((got.double() - want).abs() <= err + 2.0 ** -8 * (want.abs() + err) + 2.0 ** -25).all()
    wd = w[:, at].double().t()
    close(dx, dz @ wd, (ez + (600 + 16) * STEP * dz.abs()) @ wd.abs())
    close(dw[:, at], x.double().t() @ dz, x.double().abs().t() @ (ez + (rows + 8) * STEP * dz.abs()))
    close(db[at], dz.sum(0), (eb + (rows + 8) * STEP * dz.abs()).sum(0))
    assert not dw[:, 300:n - 300].any() and not db[300:n - 300].any()


@pytest.mark.parametrize('t, k, n', [(70000, 32768, 16), (70000, 16, 32768)])
@pytest.mark.parametrize('w_t', [False, True])
def test_weight_gradients_of_operands_past_32_bits(cuda, t, k, n, w_t):
    """x or dy of more than 2**31 values, summed over all rows; dy is 0 but in three strips, so that the sum has 210
    terms, the bound that of 210, and a strip that is lost or read elsewhere shows."""
    torch.manual_seed(k)
    at = torch.cat([torch.arange(a, a + 70) for a in (0, 65500, t - 70)]).cuda()
    x = torch.empty(t, k, device='cuda', dtype=BF).normal_()
    w = normal(n, k, scale=k ** -0.5).t() if w_t else normal(k, n, scale=k ** -0.5)
    dy = torch.zeros(t, n, device='cuda', dtype=BF)
    dy[at] = normal(210, n)
    dw, db = S.dense_matmul_backward(dy, x, w, None, bias=True)[1:]
    xs, ds = x[at].double(), dy[at].double()
    want, size = xs.t() @ ds, xs.abs().t() @ ds.abs()
    assert ((dw.double() - want).abs() <= 2.0 ** -8 * want.abs() + 1.01 * (210 + 8) * STEP * size + 2.0 ** -25).all()
    want, size = ds.sum(0), ds.abs().sum(0)
    assert ((db.double() - want).abs() <= 2.0 ** -8 * want.abs() + 1.01 * (210 + 8) * STEP * size + 2.0 ** -25).all()


def test_autograd_keeps_what_its_gradients_read(cuda):
    """Frozen weights: x is not kept and may be written again; a residual alone needs no slope."""
    x, w, b, r, dy = normal(64, 48), normal(48, 80), normal(80), normal(64, 80), normal(64, 80)
    kept = []

    def apply(*args):
        kept.clear()
        with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t.data_ptr()) or t, lambda t: t):
            return S.dense_matmul(*args, activation='silu')
    xl = x.clone().requires_grad_()
    y = apply(xl, w, b)
    assert xl.data_ptr() not in kept and len(kept) == 3     # w, the slopes, the status
    _, slope = S.dense_matmul(x, w, b, activation='silu', return_slope=True)
    want = S.dense_matmul_backward(dy, x, w, slope)
    with torch.no_grad():
        xl.zero_()
    assert torch.equal(torch.autograd.grad(y, xl, dy)[0], want[0])
    wl = w.clone().requires_grad_()
    y = apply(x, wl, b)
    assert x.data_ptr() in kept and torch.equal(torch.autograd.grad(y, wl, dy)[0], want[1])
    bl = b.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(apply(x, w, bl), bl, dy)[0],
                       S.dense_matmul_backward(dy, x, w, slope, bias=True)[2])
    rl = r.clone().requires_grad_()
    y = apply(x, w, b, rl)
    assert len(kept) == 2 and torch.equal(torch.autograd.grad(y, rl, dy)[0], dy)


def test_an_expired_wait_of_the_backward_pass_is_reported(cuda, monkeypatch):
    """A wait that nothing ends runs out in a backward pass through autograd: the product's result says so."""
    from spmm_b200 import linear as L
    x, w = normal(300, 256).requires_grad_(), normal(256, 512).requires_grad_()
    y = S.dense_matmul(x, w)
    assert S.product_status(y) == 0
    pack = L._PACK

    def short(version, dtype, act, wait_us, flags, *rest):
        return pack(version, dtype, act, 2000, flags | _lib.SPMM_CFG_EXPIRE_FIRST_WAIT, *rest)
    monkeypatch.setattr(L, '_PACK', short)
    y.backward(torch.ones_like(y), retain_graph=True)
    monkeypatch.setattr(L, '_PACK', pack)
    assert S.product_status(y) == _lib.SPMM_ETIMEOUT
    x.grad = w.grad = None
    y.backward(torch.ones_like(y))            # the word keeps what it said; the gradients are right again
    assert S.product_status(y) == _lib.SPMM_ETIMEOUT
    want = S.dense_matmul_backward(torch.ones_like(y), x.detach(), w.detach())
    assert torch.equal(x.grad, want[0]) and torch.equal(w.grad, want[1]) and S.product_status(want[0]) == 0


@pytest.mark.parametrize('rows', [1, 300, 0])
def test_a_status_that_is_kept(cuda, rows):
    x, w = normal(rows, 256), normal(256, 512)
    y = torch.empty(rows, 512, device='cuda', dtype=BF)
    for flags, want in ((_lib.LINEAR_KEEP_STATUS, 7), (0, 0)):
        status = int32(7)
        run('spmm_linear_forward', linear(rows, 256, 512, x=x, w=w, y=y, status=status, flags=flags))
        assert int(status) == want
        status, dx, dw = int32(7), torch.empty_like(x), torch.empty_like(w)
        run('spmm_linear_backward', linear(rows, 256, 512, x=x, w=w, dy=y, dx=dx, dw=dw, status=status, flags=flags))
        assert int(status) == want
