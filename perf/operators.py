"""Cases, plain forms and exact values of the dense, grouped and routed products.

Four operators: ``dense`` (``spmm_b200.dense_matmul``), ``grouped``
(``grouped_matmul``: one dense block per ragged group of rows), ``route``
(``route_topk``: expert choice, weights and the grouping of the rows) and
``combine`` (``route_combine``: the weighted sum back in token order).  A case
with ``train`` runs forward and backward.
"""

import math

import numpy as np
import torch

own = False

DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
ACTIVATIONS = ('none', 'relu', 'gelu', 'gelu_tanh', 'silu')


def _dense(name, tokens, k, n, dtype='bf16', act='none', bias=True, residual=False, train=False, w_t=False):
    return {'name': name, 'op': 'dense', 'tokens': tokens, 'k': k, 'n': n, 'dtype': dtype, 'act': act, 'bias': bias,
            'residual': residual, 'train': train, 'w_t': w_t}


def _grouped(name, tokens, experts, top, k, n, dtype='bf16', act='none', bias=False, gather=True, train=False,
             w_t=False, skew=0.0, padded=0):
    return {'name': name, 'op': 'grouped', 'tokens': tokens, 'experts': experts, 'top': top, 'k': k, 'n': n,
            'dtype': dtype, 'act': act, 'bias': bias, 'gather': gather, 'train': train, 'w_t': w_t, 'skew': skew,
            'padded': padded}


def _route(name, tokens, experts, top, dtype='fp32', scoring='softmax', renormalize=True, bias=False, train=False,
           padded=0):
    return {'name': name, 'op': 'route', 'tokens': tokens, 'experts': experts, 'top': top, 'dtype': dtype,
            'scoring': scoring, 'renormalize': renormalize, 'bias': bias, 'train': train, 'padded': padded}


def _combine(name, tokens, experts, top, n, dtype='bf16', residual=True, train=False, padded=0):
    return {'name': name, 'op': 'combine', 'tokens': tokens, 'experts': experts, 'top': top, 'n': n, 'dtype': dtype,
            'residual': residual, 'train': train, 'padded': padded}


def listed():
    return [
        # one token of a decoding step through an output projection with its residual
        _dense('dense_decode', 1, 4096, 4096, residual=True, w_t=True),
        # the tokens of a few decoding sequences, sizes that divide nothing
        _dense('dense_odd', 77, 1531, 2310, dtype='fp16', act='gelu'),
        # prefill of one long prompt through the wide product of a feed-forward layer
        _dense('dense_prefill', 8192, 4096, 16384, act='silu', bias=False, w_t=True),
        # a training micro-batch through the same kind of layer, forward and backward
        _dense('dense_train', 4096, 2048, 8192, act='gelu_tanh', residual=False, train=True),
        # a decoding batch through 64 experts: bound by the weights of the experts it touches
        _grouped('grouped_decode', 16, 64, 4, 2048, 1408, act='silu', w_t=True),
        # prefill through few wide experts, ragged, with padded tokens at the end
        _grouped('grouped_prefill', 4096, 8, 2, 4096, 4096, dtype='fp16', act='gelu', bias=True, skew=0.5, padded=37),
        # a training micro-batch through many narrow experts, popular ones among them
        _grouped('grouped_train', 8192, 64, 8, 2048, 1024, act='silu', train=True, skew=0.5),
        # rows that are in expert order already (the second product of an expert layer)
        _grouped('grouped_second', 2000, 32, 4, 1024, 2048, gather=False, w_t=True, skew=0.5),
        # routing of a decoding batch
        _route('route_decode', 32, 64, 4),
        # routing of a training micro-batch over many experts, with padded tokens
        _route('route_train', 16384, 256, 8, dtype='bf16', scoring='sigmoid', train=True, padded=100),
        # the way back of a decoding batch
        _combine('combine_decode', 32, 64, 4, 2048),
        # the way back of a training micro-batch, forward and backward
        _combine('combine_train', 16384, 64, 8, 2048, train=True, padded=100),
    ]


def _size(rng, lo, hi):
    """Log-uniform; three in four rounded to a multiple of 64 where that leaves the range, the rest any whole number."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, v // 64 * 64) if v >= 64 and rng.random() < 0.75 else v


def draw(rng):
    op = rng.choice(['dense', 'grouped', 'grouped', 'route', 'combine', 'dense'])
    dtype = rng.choice(['bf16', 'bf16', 'fp16'])
    train = rng.random() < 0.5
    tokens = int(round(math.exp(rng.uniform(0.0, math.log(8192)))))
    while op == 'dense':
        case = _dense('', tokens, _size(rng, 64, 8192), _size(rng, 64, 8192), dtype, rng.choice(ACTIVATIONS),
                      rng.random() < 0.5, rng.random() < 0.5, train, rng.random() < 0.5)
        if work(case)['flops'] <= 1e12:
            return case
    experts, top = rng.choice([(8, 2), (16, 2), (32, 4), (64, 4), (64, 6), (64, 8), (128, 8)])
    while op == 'grouped':
        case = _grouped('', tokens, experts, top, _size(rng, 128, 4096), _size(rng, 128, 4096), dtype,
                        rng.choice(ACTIVATIONS), rng.random() < 0.5, rng.random() < 0.5, train, rng.random() < 0.5,
                        rng.choice([0.0, 0.5]), tokens // 16 if rng.random() < 0.5 else 0)
        if work(case)['flops'] <= 8e11 and experts * case['k'] * case['n'] <= 1 << 28:
            return case
    if op == 'route':
        experts = rng.choice([8, 60, 64, 128, 160, 256, 512])
        return _route('', tokens, experts, rng.randint(1, 8), rng.choice(['fp32', 'bf16', 'fp16']),
                      rng.choice(['softmax', 'sigmoid']), rng.random() < 0.5, rng.random() < 0.5, train,
                      tokens // 16 if rng.random() < 0.5 else 0)
    return _combine('', tokens, experts, top, _size(rng, 64, 4096), dtype, rng.random() < 0.5, train,
                    tokens // 16 if rng.random() < 0.5 else 0)


def _logits(case, g, skew=0.0):
    """Router scores: a normal part per token and, with ``skew``, a popularity per expert; padded tokens (at the
    end) are masked whole."""
    tokens, experts = case['tokens'], case['experts']
    logits = torch.randn(tokens, experts, device='cuda', generator=g)
    if skew:
        logits += skew * torch.randn(experts, device='cuda', generator=g)
    if case['padded']:
        logits[tokens - case['padded']:] = -math.inf
    return logits


def _grouping(experts_of, experts):
    """offsets [E+1], rows [T k] (-1 behind the last group) and slots [T,k] of the choices [T,k] (-1: none)."""
    tokens, top = experts_of.shape
    flat = experts_of.reshape(-1).long()
    chosen = flat >= 0
    order = torch.sort(torch.where(chosen, flat, experts), stable=True).indices
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel(), device=order.device)
    slots = torch.where(chosen, place, -1).reshape(tokens, top).int()
    rows = torch.where(chosen[order], order // top, -1).int()
    ids = torch.arange(experts + 1, device=flat.device)
    offsets = (chosen[None, :] & (flat[None, :] < ids[:, None])).sum(1).int()
    return offsets, rows, slots


def _choices(logits, top, bias=None):
    """The ``top`` best experts of each token, best first, ties to the lowest index; -1 where nothing is left."""
    key = logits.float()
    key = torch.where(torch.isnan(key), -math.inf, key)
    if bias is not None:
        key = key + bias
    best, index = torch.sort(key, dim=1, descending=True, stable=True)
    return torch.where(best[:, :top] > -math.inf, index[:, :top], -1)


def prepare(case, seed):
    g = torch.Generator(device='cuda')
    g.manual_seed(int(seed) * 7919 + 17)
    dt = DTYPES[case['dtype']]

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, device='cuda', generator=g) * scale).to(dtype)

    s = {'case': case}
    op = case['op']
    if op == 'dense':
        t, k, n = case['tokens'], case['k'], case['n']
        s['x'] = normal(t, k)
        s['w'] = normal(n, k, scale=k ** -0.5).t() if case['w_t'] else normal(k, n, scale=k ** -0.5)
        s['bias'] = normal(n) if case['bias'] else None
        s['residual'] = normal(t, n) if case['residual'] else None
        s['dy'] = normal(t, n) if case['train'] else None
        return s
    e, top, t = case['experts'], case['top'], case['tokens']
    if op == 'route':
        s['logits'] = _logits(case, g).to(dt)
        s['bias'] = normal(e, scale=0.1, dtype=torch.float32) if case['bias'] else None
        s['dweights'] = normal(t, top, dtype=torch.float32) if case['train'] else None
        return s
    logits = _logits(case, g, case.get('skew', 0.0))
    s['experts'] = _choices(logits, top).int()
    s['offsets'], s['rows'], s['slots'] = _grouping(s['experts'], e)
    if op == 'grouped':
        k, n = case['k'], case['n']
        s['x'] = normal(t if case['gather'] else t * top, k)
        s['w'] = normal(e, n, k, scale=k ** -0.5).transpose(1, 2) if case['w_t'] else normal(e, k, n, scale=k ** -0.5)
        s['bias'] = normal(e, n) if case['bias'] else None
        s['dy'] = normal(t * top, n) if case['train'] else None
        # a plain program pads its groups to the longest one, which it knows from making them
        s['longest'] = int((s['offsets'][1:] - s['offsets'][:-1]).max())
        return s
    s['y'] = normal(t * top, case['n'])
    s['weights'] = torch.softmax(normal(t, top, dtype=torch.float32), 1)
    s['residual'] = normal(t, case['n']) if case['residual'] else None
    s['dout'] = normal(t, case['n']) if case['train'] else None
    return s


# ---- plain forms ------------------------------------------------------------

def _act(z, name):
    """The activation and its derivative."""
    if name == 'none':
        return z, torch.ones_like(z)
    if name == 'relu':
        return torch.where(z > 0, z, 0.0), (z > 0).to(z.dtype)
    if name == 'silu':
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    if name == 'gelu':
        cdf = 0.5 * (1 + torch.erf(z * 0.5 ** 0.5))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    c = (2 / math.pi) ** 0.5
    th = torch.tanh(c * (z + 0.044715 * z * z * z))
    return 0.5 * z * (1 + th), 0.5 * (1 + th) + 0.5 * z * (1 - th * th) * c * (1 + 3 * 0.044715 * z * z)


def _plain_dense(s, c):
    dt = DTYPES[c['dtype']]
    x, w = s['x'].float(), s['w'].float()
    z = x @ w
    if s['bias'] is not None:
        z = z + s['bias'].float()
    a, slope = _act(z, c['act'])
    out = {'y': (a if s['residual'] is None else a + s['residual'].float()).to(dt)}
    if c['train']:
        dz = s['dy'].float() * slope
        out['dx'] = (dz @ w.t()).to(dt)
        out['dw'] = (x.t() @ dz).to(dt)
        if s['bias'] is not None:
            out['dbias'] = dz.sum(0).to(dt)
    return out


def _plain_grouped(s, c):
    """Each group's rows padded to the longest group, one batched product over the groups."""
    dt = DTYPES[c['dtype']]
    e, longest = c['experts'], s['longest']
    total = c['tokens'] * c['top']
    offsets = s['offsets'].long()
    place = torch.arange(longest, device='cuda')[None, :] + offsets[:-1, None]      # [E, longest]
    inside = place < offsets[1:, None]
    place = torch.where(inside, place, 0)
    token = s['rows'].long()[place] if c['gather'] else place
    token = torch.where(inside, token, 0)
    keep = inside[:, :, None]
    x = torch.where(keep, s['x'].float()[token], 0.0)
    w = s['w'].float()
    z = torch.bmm(x, w)
    if s['bias'] is not None:
        z = z + s['bias'].float()[:, None, :]
    a, slope = _act(z, c['act'])
    back = torch.where(inside, place, total)                                        # padding goes to a spare row
    y = torch.zeros(total + 1, c['n'], device='cuda')
    y[back] = torch.where(keep, a, 0.0)
    y[total] = 0
    out = {'y': y[:total].to(dt)}
    if c['train']:
        dz = torch.where(keep, s['dy'].float()[place] * slope, 0.0)
        out['dw'] = torch.bmm(x.transpose(1, 2), dz).to(dt)
        dx = torch.zeros(total + 1, c['k'], device='cuda')
        dx[back] = torch.bmm(dz, w.transpose(1, 2))
        dx[total] = 0
        if c['gather']:
            slots = s['slots'].long()
            dx = dx[torch.where(slots >= 0, slots, total)].sum(1)
        else:
            dx = dx[:total]
        out['dx'] = dx.to(dt)
        if s['bias'] is not None:
            out['dbias'] = dz.sum(1).to(dt)
    return out


def _plain_route(s, c):
    logits = s['logits'].float()
    index = _choices(s['logits'], c['top'], s['bias'])
    offsets, rows, slots = _grouping(index, c['experts'])
    chosen = index >= 0
    at = torch.where(chosen, index, 0)
    if c['scoring'] == 'softmax':
        top = logits.max(1, keepdim=True).values
        p = torch.exp(logits - torch.where(top > -math.inf, top, 0.0))
        total = p.sum(1, keepdim=True)
        p = p / torch.where(total > 0, total, 1.0)
    else:
        p = 1 / (1 + torch.exp(-logits))
    sel = torch.where(chosen, p.gather(1, at), 0.0)
    norm = sel.sum(1, keepdim=True)
    norm = torch.where(norm > 0, norm, 1.0)
    weights = sel / norm if c['renormalize'] else sel
    out = {'weights': weights, 'experts': index.int(), 'offsets': offsets, 'rows': rows, 'slots': slots}
    if c['train']:
        d = torch.where(chosen, s['dweights'], 0.0)
        if c['renormalize']:
            d = (d - (d * weights).sum(1, keepdim=True)) / norm
        if c['scoring'] == 'softmax':
            dp = torch.zeros_like(p).scatter_add_(1, at, torch.where(chosen, d, 0.0))
            grad = p * (dp - (d * sel).sum(1, keepdim=True))
        else:
            grad = torch.zeros_like(p).scatter_add_(1, at, torch.where(chosen, d * sel * (1 - sel), 0.0))
        out['dlogits'] = grad.to(s['logits'].dtype)
    return out


def _plain_combine(s, c):
    dt = DTYPES[c['dtype']]
    slots = s['slots'].long()
    chosen = (slots >= 0)[:, :, None]
    picked = torch.where(chosen, s['y'].float()[torch.where(slots >= 0, slots, 0)], 0.0)
    o = (picked * s['weights'][:, :, None]).sum(1)
    out = {'out': (o if s['residual'] is None else o + s['residual'].float()).to(dt)}
    if c['train']:
        d = s['dout'].float()
        out['dweights'] = (picked * d[:, None, :]).sum(2)
        dy = torch.zeros(c['tokens'] * c['top'] + 1, c['n'], device='cuda')
        dy[torch.where(slots >= 0, slots, c['tokens'] * c['top'])] = s['weights'][:, :, None] * d[:, None, :]
        out['dy'] = dy[:-1].to(dt)
    return out


# ---- the framework's calls --------------------------------------------------

def _own_run(s, c):
    import spmm_b200 as S
    op = c['op']
    if op == 'dense':
        if not c['train']:
            return {'y': S.dense_matmul(s['x'], s['w'], s['bias'], s['residual'], activation=c['act'])}
        y, slope = S.dense_matmul(s['x'], s['w'], s['bias'], s['residual'], activation=c['act'], return_slope=True)
        dx, dw, db = S.dense_matmul_backward(s['dy'], s['x'], s['w'], slope, bias=s['bias'] is not None)
        out = {'y': y, 'dx': dx, 'dw': dw}
        return out if db is None else {**out, 'dbias': db}
    if op == 'route':
        weights, r = S.route_topk(s['logits'], c['top'], scoring=c['scoring'], renormalize=c['renormalize'],
                                  bias=s['bias'])
        out = {'weights': weights, 'experts': r.experts, 'offsets': r.offsets, 'rows': r.rows, 'slots': r.slots}
        if c['train']:
            out['dlogits'] = S.route_topk_backward(s['dweights'], s['logits'], r, scoring=c['scoring'],
                                                   renormalize=c['renormalize'])
        return out
    r = S.Routing(s['experts'], s['slots'], s['rows'], s['offsets'])
    if op == 'grouped':
        if not c['train']:
            return {'y': S.grouped_matmul(s['x'], s['w'], r, s['bias'], activation=c['act'], gather=c['gather'])}
        y, slope = S.grouped_matmul(s['x'], s['w'], r, s['bias'], activation=c['act'], gather=c['gather'],
                                    return_slope=True)
        dx, dw, db = S.grouped_matmul_backward(s['dy'], s['x'], s['w'], r, slope, gather=c['gather'],
                                               bias=s['bias'] is not None)
        out = {'y': y, 'dx': dx, 'dw': dw}
        return out if db is None else {**out, 'dbias': db}
    out = {'out': S.route_combine(s['y'], r, s['weights'], s['residual'])}
    if c['train']:
        out['dy'], out['dweights'] = S.route_combine_backward(s['dout'], s['y'], r, s['weights'])
    return out


def run(state):
    c = state['case']
    if own:
        return _own_run(state, c)
    return {'dense': _plain_dense, 'grouped': _plain_grouped, 'route': _plain_route,
            'combine': _plain_combine}[c['op']](state, c)


# ---- what a pass cannot do without ------------------------------------------

def work(case):
    c, size = case, {'bf16': 2, 'fp16': 2, 'fp32': 4}[case['dtype']]
    t = c['tokens']
    live = t - c.get('padded', 0)
    if c['op'] == 'dense':
        k, n = c['k'], c['n']
        forward = size * (t * k + k * n + t * n + (n if c['bias'] else 0) + (t * n if c['residual'] else 0))
        # backward: dy, x and w are read, dx, dw and the bias gradient written (x and w read once for both directions)
        backward = size * (t * n + t * k + k * n + (n if c['bias'] else 0))
        return {'bytes': forward + (backward if c['train'] else 0), 'flops': 2 * t * k * n * (3 if c['train'] else 1)}
    e, top = c['experts'], c['top']
    total, used = t * top, live * top
    if c['op'] == 'grouped':
        k, n = c['k'], c['n']
        touched = e * (1 - (1 - top / e) ** live)       # experts that at least one token chose, evenly spread
        xs = (live if c['gather'] else used) * k
        forward = size * (xs + touched * k * n + total * n + (touched * n if c['bias'] else 0)) + 4 * (e + 1 + total)
        backward = size * (used * n + (t if c['gather'] else total) * k + e * k * n + (e * n if c['bias'] else 0))
        return {'bytes': int(forward + (backward if c['train'] else 0)),
                'flops': 2 * used * k * n * (3 if c['train'] else 1)}
    if c['op'] == 'route':
        forward = size * t * e + 4 * (4 * total + e + 1) + (4 * e if c['bias'] else 0)
        backward = 4 * total + size * t * e
        return {'bytes': forward + (backward if c['train'] else 0), 'flops': (8 if c['train'] else 5) * t * e}
    n = c['n']
    forward = size * (used * n + t * n + (t * n if c['residual'] else 0)) + 8 * total
    backward = size * (t * n + total * n) + 4 * total
    return {'bytes': forward + (backward if c['train'] else 0), 'flops': (5 if c['train'] else 2) * used * n}


# ---- exact values, by the definitions in 64 bits ------------------------------

def _act_exact(z, name):
    """Activation values and derivatives in 64 bits, the derivative by its own closed form."""
    if name == 'none':
        return z, None
    if name == 'relu':
        return z.clamp(min=0), (z > 0).double()
    if name == 'silu':
        s = torch.sigmoid(z)
        return z * s, s + z * s * torch.sigmoid(-z)
    if name == 'gelu':
        upper = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        return z * upper, upper + z * torch.exp(-z.square() / 2) / math.sqrt(2 * math.pi)
    u = math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
    s = torch.sigmoid(2 * u)                              # (1 + tanh u) / 2
    return z * s, s + z * 2 * s * torch.sigmoid(-2 * u) * math.sqrt(2 / math.pi) * (1 + 0.134145 * z.square())


def exact(case, seed):
    c, s = case, prepare(case, seed)
    op = c['op']
    if op == 'dense':
        x, w = s['x'].double(), s['w'].double()
        z = torch.matmul(x, w)
        if s['bias'] is not None:
            z += s['bias'].double()
        y, slope = _act_exact(z, c['act'])
        out = {'y': y if s['residual'] is None else y + s['residual'].double()}
        if c['train']:
            dz = s['dy'].double()
            dz = dz if slope is None else dz * slope
            out['dx'], out['dw'] = torch.einsum('tn,kn->tk', dz, w), torch.einsum('tk,tn->kn', x, dz)
            if s['bias'] is not None:
                out['dbias'] = torch.einsum('tn->n', dz)
        return out
    t, top, e = c['tokens'], c['top'], c['experts']
    if op == 'grouped':
        ends = s['offsets'].tolist()
        x, k, n = s['x'], c['k'], c['n']
        out = {'y': torch.zeros(t * top, n, dtype=torch.float64, device='cuda')}
        if c['train']:
            out['dx'] = torch.zeros(x.shape[0], k, dtype=torch.float64, device='cuda')
            out['dw'] = torch.zeros(e, k, n, dtype=torch.float64, device='cuda')
            if s['bias'] is not None:
                out['dbias'] = torch.zeros(e, n, dtype=torch.float64, device='cuda')
        for i in range(e):
            a, b = ends[i], ends[i + 1]
            if a == b:
                continue
            at = s['rows'][a:b].long() if c['gather'] else torch.arange(a, b, device='cuda')
            xi, wi = x[at].double(), s['w'][i].double()
            z = xi @ wi
            if s['bias'] is not None:
                z += s['bias'][i].double()
            out['y'][a:b], slope = _act_exact(z, c['act'])
            if c['train']:
                dz = s['dy'][a:b].double()
                dz = dz if slope is None else dz * slope
                out['dx'].index_add_(0, at, dz @ wi.t())
                out['dw'][i] = xi.t() @ dz
                if s['bias'] is not None:
                    out['dbias'][i] = dz.sum(0)
        return out
    if op == 'route':
        return _exact_route(s, c)
    slots, w = s['slots'].cpu().numpy(), s['weights'].double()
    out = {'out': torch.zeros(t, c['n'], dtype=torch.float64, device='cuda')}
    if s['residual'] is not None:
        out['out'] += s['residual'].double()
    if c['train']:
        out['dweights'] = torch.zeros(t, top, dtype=torch.float64, device='cuda')
        out['dy'] = torch.zeros(t * top, c['n'], dtype=torch.float64, device='cuda')
    for j in range(top):
        live = torch.from_numpy(np.flatnonzero(slots[:, j] >= 0)).cuda()
        at = torch.from_numpy(slots[slots[:, j] >= 0, j].astype(np.int64)).cuda()
        yj = s['y'][at].double()
        out['out'][live] += w[live, j, None] * yj
        if c['train']:
            dj = s['dout'][live].double()
            out['dweights'][live, j] = (yj * dj).sum(1)
            out['dy'][at] = w[live, j, None] * dj
    return out


def _exact_route(s, c):
    """numpy, from the definition: the choice goes by the 32-bit sum of logit and bias, the weights by 64 bits."""
    t, top, e = c['tokens'], c['top'], c['experts']
    score = s['logits'].float().cpu().numpy()
    key = score if s['bias'] is None else score + s['bias'].cpu().numpy()
    order = np.lexsort((np.broadcast_to(np.arange(e), key.shape), -key), axis=1)[:, :top]
    ok = np.take_along_axis(key, order, 1) > -np.inf
    experts = np.where(ok, order, -1)
    flat = experts.reshape(-1)
    live = np.flatnonzero(flat >= 0)
    live = live[np.lexsort((live, flat[live]))]
    rows = np.full(t * top, -1, np.int32)
    rows[:live.size] = live // top
    slots = np.full(t * top, -1, np.int32)
    slots[live] = np.arange(live.size)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat[live], minlength=e))]).astype(np.int32)
    z = score.astype(np.float64)
    with np.errstate(invalid='ignore', over='ignore'):
        if c['scoring'] == 'softmax':
            m = z.max(1, keepdims=True)
            p = np.exp(z - np.where(np.isfinite(m), m, 0))
            p /= np.maximum(p.sum(1, keepdims=True), 1e-300)
        else:
            p = 0.5 * (1 + np.tanh(z / 2))
    picked = np.where(ok, np.take_along_axis(p, order, 1), 0)
    norm = picked.sum(1, keepdims=True)
    norm = np.where(norm > 0, norm, 1)
    weights = picked / norm if c['renormalize'] else picked
    out = {'weights': weights, 'experts': experts.astype(np.int32), 'offsets': offsets, 'rows': rows,
           'slots': slots.reshape(t, top)}
    if c['train']:
        d = np.where(ok, s['dweights'].double().cpu().numpy(), 0)
        if c['renormalize']:                      # weights_j = p_j / sum p: d p_j = (d_j - <d, weights>) / sum p
            d = np.where(ok, d - (d * weights).sum(1, keepdims=True), 0) / norm
        dp = np.zeros_like(p)
        np.put_along_axis(dp, order, d, 1)        # `order` holds different experts in a row
        if c['scoring'] == 'softmax':
            out['dlogits'] = p * (dp - (dp * p).sum(1, keepdims=True))
        else:
            out['dlogits'] = dp * p * (1 - p)
    return {k: torch.from_numpy(np.ascontiguousarray(v)) for k, v in out.items()}
