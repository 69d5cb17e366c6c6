"""Cases that measure the normalisation and orthogonalised-update operators, with their plain forms.

Operators: layer norm over the rows of a hidden layer (``norm``), its backward pass with the reduction of the parameter
gradients (``norm_grad``), the backward of that backward pass, which a critic under a gradient penalty needs
(``norm_grad2``), the Newton-Schulz orthogonalisation of an update (``orth``) and the optimizer step built on it
(``muon``).  ``own`` False: elementary torch operations; True: this package's kernels.
"""
import math

import torch

own = False

_COEF = (3.4445, -4.7750, 2.0315)
_STEPS, _ORTH_EPS, _EPS = 5, 1e-7, 1e-3
_TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16}


def listed():
    return [
        # one hidden layer at the default training batch: latency
        dict(name='norm_hidden_b32', kind='norm', rows=32, width=256, dtype='f32', slope=0.0, pad=False),
        # prediction of a whole data set (the 100000-sample evaluation): one hidden layer
        dict(name='norm_predict_100k', kind='norm', rows=100000, width=256, dtype='f32', slope=0.0, pad=False),
        # rows of all E. coli genes (odd width, rows padded to 16 bytes as the package lays them out), 16-bit storage
        dict(name='norm_genes_bf16', kind='norm', rows=4096, width=4297, dtype='bf16', slope=0.2, pad=True),
        # critic step at 512 rows: the stacked [real; fake; interpolated] rows of a hidden layer
        dict(name='norm_grad_critic_b512', kind='norm_grad', rows=1536, width=256, dtype='f32', slope=0.0, pad=False),
        # wide layers over many rows, 16-bit storage
        dict(name='norm_grad_large_bf16', kind='norm_grad', rows=40000, width=1000, dtype='bf16', slope=0.2, pad=False),
        # penalty's second order on the interpolated rows at 512
        dict(name='norm_grad2_b512', kind='norm_grad2', rows=512, width=256, dtype='f32', slope=0.0, pad=False),
        # the same over wide rows (odd width, unpadded)
        dict(name='norm_grad2_wide', kind='norm_grad2', rows=8192, width=1077, dtype='f32', slope=0.2, pad=False),
        # a hidden kernel: latency of the product chain
        dict(name='orth_hidden_256', kind='orth', rows=256, cols=256, dtype='f32', seen=640),
        # the GTEx-shaped critic's first kernel (genes and covariates by hidden width)
        dict(name='orth_critic_in', kind='orth', rows=18161, cols=256, dtype='f32', seen=1920),
        # a wide output kernel of a 1000-wide generator, 16-bit storage
        dict(name='orth_wide_bf16', kind='orth', rows=1000, cols=4297, dtype='bf16', seen=1920),
        # optimizer step over all kernels of the E. coli-shaped critic and of the GTEx-shaped generator
        dict(name='muon_ecoli_critic', kind='muon', d0=4318, d1=128, d2=128, d3=0, seen=640, decay=0.0, nesterov=True),
        dict(name='muon_gtex_generator', kind='muon', d0=71, d1=256, d2=256, d3=18154, seen=640, decay=0.01, nesterov=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(['norm', 'norm_grad', 'norm_grad2', 'orth', 'muon'])
    if kind in ('norm', 'norm_grad', 'norm_grad2'):
        rows, width = _log(rng, 1, 100000), _log(rng, 8, 18154)
        most = {'norm': 25000000, 'norm_grad': 16000000, 'norm_grad2': 8800000}[kind]
        rows = max(1, min(rows, most // width))
        return dict(kind=kind, rows=rows, width=width, dtype=rng.choice(['f32', 'bf16']), slope=rng.choice([0.0, 0.2]),
                    pad=rng.random() < 0.5)
    if kind == 'orth':
        n = _log(rng, 16, 1024)
        m = max(n, min(_log(rng, 16, 18161), 4600000 // n))
        while 3.0 * m * n * n + 15.0 * n ** 3 > 2.6e10:
            m, n = max(16, m * 3 // 4), max(16, min(n * 3 // 4, m * 3 // 4))
        rows, cols = (m, n) if rng.random() < 0.5 else (n, m)
        return dict(kind='orth', rows=rows, cols=cols, dtype=rng.choice(['f32', 'bf16']), seen=_log(rng, 64, 1920))
    d0, d1, d2 = _log(rng, 16, 18161), _log(rng, 16, 256), _log(rng, 16, 256)
    d3 = rng.choice([0, _log(rng, 16, 18154)])
    return dict(kind='muon', d0=d0, d1=d1, d2=d2, d3=d3, seen=_log(rng, 64, 1920), decay=rng.choice([0.0, 0.01]),
                nesterov=rng.random() < 0.7)


def _gen(seed):
    g = torch.Generator(device='cuda')
    g.manual_seed(int(seed))
    return g


def _rand(g, *shape):
    return torch.randn(*shape, generator=g, device='cuda')


def _place(v, dtype, pad):
    """`v` in the case's type, in rows padded to a multiple of 4 elements where `pad`."""
    width = v.shape[1]
    t = torch.zeros(v.shape[0], (width + 3) & ~3 if pad else width, device='cuda', dtype=dtype)[:, :width]
    t.copy_(v)
    return t


def _rows(g, rows, width, dtype, pad, center=None):
    v = _rand(g, rows, width)
    return _place(v if center is None else v + center, dtype, pad)


def _update(g, rows, cols, seen):
    """A kernel's accumulated gradient: `seen` samples of correlated inputs against sparse deltas, older ones decayed."""
    a = _rand(g, seen, 8) @ _rand(g, 8, rows) / math.sqrt(8.0) + 0.5 * _rand(g, seen, rows)
    d = torch.relu(_rand(g, seen, cols)) * torch.exp(0.5 * _rand(g, cols)) * torch.sign(_rand(g, seen, 1))
    age = torch.arange(seen, device='cuda', dtype=torch.float32)[:, None] / seen
    return a.t().contiguous() @ (d * torch.exp(-3.0 * age)) * (1.0 / seen)


def _shapes(case):
    s = [(case['d0'], case['d1']), (case['d1'], case['d2'])]
    return s + [(case['d2'], case['d3'])] if case['d3'] else s


def _act(n, slope):
    return torch.where(n > 0, n, slope * n)


def prepare(case, seed):
    g = _gen(seed)
    c = dict(case)
    if c['kind'] in ('norm', 'norm_grad', 'norm_grad2'):
        rows, width, dt = c['rows'], c['width'], _TYPES[c['dtype']]
        c['gamma'] = 1.0 + 0.2 * _rand(g, width)
        c['beta'] = 0.2 * _rand(g, width)
        c['x'] = _rows(g, rows, width, dt, c['pad'], center=0.5 + 0.5 * _rand(g, width))   # a Dense layer's output with its bias
        if c['kind'] != 'norm':
            x = c['x'].float()                       # what the forward pass left
            c['mean'] = x.mean(1)
            xc = x - c['mean'][:, None]
            c['rstd'] = torch.rsqrt((xc * xc).mean(1) + _EPS)
            c['y'] = _place(_act(xc * c['rstd'][:, None] * c['gamma'] + c['beta'], c['slope']), dt, c['pad'])
            c['dy'] = _rows(g, rows, width, dt, c['pad'])
        if c['kind'] == 'norm_grad2':
            c['u'] = _rows(g, rows, width, dt, c['pad'])
    elif c['kind'] == 'orth':
        c['x'] = _update(g, c['rows'], c['cols'], c['seen']).to(_TYPES[c['dtype']])
    else:
        c['w'], c['g'], c['m'] = [], [], []
        for r, k in _shapes(c):
            lim = math.sqrt(6.0 / (r + k))
            c['w'].append((torch.rand(r, k, generator=g, device='cuda') * 2 - 1) * lim)
            c['g'].append(_update(g, r, k, c['seen']))
            c['m'].append(5.0 * _update(g, r, k, c['seen']))
    return c


# ---- plain forms ----

def _norm(s):
    x = s['x'].float()
    mean = x.mean(1)
    xc = x - mean[:, None]
    rstd = torch.rsqrt((xc * xc).mean(1) + _EPS)
    y = _act(xc * rstd[:, None] * s['gamma'] + s['beta'], s['slope'])
    return y.to(s['x'].dtype), mean, rstd


def _norm_grad(s):
    x, dy, r = s['x'].float(), s['dy'].float(), s['rstd'][:, None]
    h = (x - s['mean'][:, None]) * r
    dn = torch.where(s['y'] > 0, dy, s['slope'] * dy)
    gr = dn * s['gamma']
    dx = r * (gr - gr.mean(1, keepdim=True) - h * (gr * h).mean(1, keepdim=True))
    return dx.to(s['x'].dtype), (dn * h).sum(0), dn.sum(0)


def _norm_grad2(s):
    x, dy, u, r = s['x'].float(), s['dy'].float(), s['u'].float(), s['rstd'][:, None]
    h = (x - s['mean'][:, None]) * r
    up = s['y'] > 0
    dn = torch.where(up, dy, s['slope'] * dy)
    gr = dn * s['gamma']
    mg, mu = gr.mean(1, keepdim=True), u.mean(1, keepdim=True)
    cg, cu = (gr * h).mean(1, keepdim=True), (u * h).mean(1, keepdim=True)
    q = r * (u - mu - h * cu)
    ddy = s['gamma'] * q
    ddy = torch.where(up, ddy, s['slope'] * ddy)
    dx = r * r * (h * (3 * cg * cu + mg * mu - (gr * u).mean(1, keepdim=True)) - cu * (gr - mg) - cg * (u - mu))
    return ddy.to(s['x'].dtype), dx.to(s['x'].dtype), (dn * q).sum(0)


def _orth(x):
    a, b, c = _COEF
    x = x.float()
    x = x / (torch.sqrt((x * x).sum()) + _ORTH_EPS)
    tall = x.shape[0] > x.shape[1]
    for _ in range(_STEPS):
        if tall:
            A = x.t() @ x
            x = a * x + x @ (b * A + c * (A @ A))
        else:
            A = x @ x.t()
            x = a * x + (b * A + c * (A @ A)) @ x
    return x


def _muon(s, lr=0.02, momentum=0.95):
    for w, g, m in zip(s['w'], s['g'], s['m']):
        m.mul_(momentum).add_(g)
        o = _orth(g + momentum * m if s['nesterov'] else m)
        w.mul_(1.0 - lr * s['decay']).sub_(o * (lr * math.sqrt(max(1.0, w.shape[1] / w.shape[0]))))
    return s['w'], s['m']


def run(state):
    s = state
    if own:
        from adversarial_gene_expression_amd import ops
        if s['kind'] == 'norm':
            return ops.layer_norm(s['x'], s['gamma'], s['beta'], eps=_EPS, act=1, slope=s['slope'])
        if s['kind'] == 'norm_grad':
            return ops.layer_norm_backward(s['dy'], s['x'], s['mean'], s['rstd'], s['gamma'], y=s['y'], act=1, slope=s['slope'])
        if s['kind'] == 'norm_grad2':
            return ops.layer_norm_backward2(s['u'], s['dy'], s['x'], s['mean'], s['rstd'], s['gamma'], y=s['y'], act=1,
                                            slope=s['slope'])
        if s['kind'] == 'orth':
            return ops.orthogonalize(s['x'], steps=_STEPS, coefficients=_COEF, eps=_ORTH_EPS)
        ops.muon(s['w'], s['g'], s['m'], 0.02, momentum=0.95, nesterov=s['nesterov'], weight_decay=s['decay'], steps=_STEPS,
                 coefficients=_COEF, eps=_ORTH_EPS)
        return s['w'], s['m']
    if s['kind'] == 'orth':
        return _orth(s['x']).to(s['x'].dtype)
    return {'norm': _norm, 'norm_grad': _norm_grad, 'norm_grad2': _norm_grad2, 'muon': _muon}[s['kind']](s)


def work(case):
    if case['kind'] in ('norm', 'norm_grad', 'norm_grad2'):
        e = float(case['rows']) * case['width']
        b = 4 if case['dtype'] == 'f32' else 2
        arrays, params, flops = {'norm': (2, 2, 8), 'norm_grad': (4, 3, 14), 'norm_grad2': (6, 2, 30)}[case['kind']]
        return {'bytes': arrays * e * b + 8.0 * case['rows'] + 4.0 * params * case['width'], 'flops': flops * e}

    def products(r, c):
        m, n = float(max(r, c)), float(min(r, c))
        # one symmetric product over the long side, one product back, and three symmetric products of the short side a step
        return 3.0 * m * n * n + _STEPS * 3.0 * n ** 3

    if case['kind'] == 'orth':
        b = 4 if case['dtype'] == 'f32' else 2
        return {'bytes': 2.0 * b * case['rows'] * case['cols'], 'flops': products(case['rows'], case['cols'])}
    return {'bytes': sum(20.0 * r * c for r, c in _shapes(case)), 'flops': sum(products(r, c) for r, c in _shapes(case))}


# ---- 64 bits: the forward definition differentiated by torch, and the iteration in Horner's form ----

def _exact_forward(x, gamma, beta, mask, slope):
    d = x - torch.sum(x, 1, keepdim=True) / x.shape[1]
    n = gamma * d / torch.sqrt(torch.sum(d ** 2, 1, keepdim=True) / x.shape[1] + _EPS) + beta
    return n * torch.where(mask if mask is not None else n > 0, 1.0, slope)


def _exact_orth(x):
    a, b, c = _COEF
    x = x / (torch.linalg.vector_norm(x) + _ORTH_EPS)
    if x.shape[0] < x.shape[1]:
        return _exact_orth_tall(x.t().contiguous(), a, b, c).t()
    return _exact_orth_tall(x, a, b, c)


def _exact_orth_tall(x, a, b, c):
    one = torch.eye(x.shape[1], dtype=x.dtype, device=x.device)
    for _ in range(_STEPS):
        A = x.t().contiguous() @ x
        x = x @ (a * one + A @ (b * one + c * A))
    return x


def exact(case, seed):
    s = prepare(case, seed)
    up = lambda t: t.to(torch.float64)  # noqa: E731
    if s['kind'] == 'norm':
        x = up(s['x'])
        d = x - torch.sum(x, 1, keepdim=True) / x.shape[1]
        return (_exact_forward(x, up(s['gamma']), up(s['beta']), None, s['slope']), torch.sum(x, 1) / x.shape[1],
                1 / torch.sqrt(torch.sum(d ** 2, 1) / x.shape[1] + _EPS))
    if s['kind'] in ('norm_grad', 'norm_grad2'):
        second = s['kind'] == 'norm_grad2'
        x, gamma, beta, dy = (up(s[k]).requires_grad_(True) for k in ('x', 'gamma', 'beta', 'dy'))
        n = _exact_forward(x, gamma, beta, s['y'] > 0, s['slope'])
        if not second:
            return torch.autograd.grad(n, (x, gamma, beta), dy)
        dx, = torch.autograd.grad(n, x, dy, create_graph=True)
        return torch.autograd.grad(dx, (dy, x, gamma), up(s['u']))
    if s['kind'] == 'orth':
        return _exact_orth(up(s['x']))
    ws, ms = [], []
    for w, g, m in zip(s['w'], s['g'], s['m']):
        m2 = 0.95 * up(m) + up(g)
        u = up(g) + 0.95 * m2 if s['nesterov'] else m2
        ms.append(m2)
        ws.append((1 - 0.02 * s['decay']) * up(w) - 0.02 * max(1.0, w.shape[1] / w.shape[0]) ** 0.5 * _exact_orth(u))
    return ws, ms
