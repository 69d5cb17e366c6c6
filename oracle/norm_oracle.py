"""Layer normalisation and its two backward passes, the Newton-Schulz orthogonalisation and the Muon step, in float64 on
the CPU (test infrastructure only).  No reference counterpart: tf_utils.py:85-88 has no normalisation and
tf_utils.py:285-288 only RMSprop / Adam.  `*_size` functions return, per element, the sum of the absolute values of the
terms the result is made of: a rounding error is a small multiple of it."""
import math

import torch


def t64(a):
    return torch.as_tensor(a).detach().to('cpu', torch.float64)


def act(n, slope, on):
    return torch.where(n > 0, n, slope * n) if on else n


def forward(x, gamma, beta, eps, slope=0.0, on=0):
    mean = x.mean(1)
    d = x - mean[:, None]
    rstd = 1.0 / torch.sqrt((d * d).mean(1) + eps)
    return act(gamma * d * rstd[:, None] + beta, slope, on), mean, rstd


def forward_size(x, gamma, beta, rstd):
    ax = x.abs()
    return gamma.abs() * (ax + ax.mean(1, keepdim=True)) * rstd[:, None] + beta.abs()


def _parts(dy, x, mean, rstd, y, slope, on):
    h = (x - mean[:, None]) * rstd[:, None]
    dn = torch.where(y > 0, dy, slope * dy) if on else dy
    return h, dn, (x.abs() + mean.abs()[:, None]) * rstd[:, None]


def _m(t):
    return t.mean(1, keepdim=True)


def backward(dy, x, mean, rstd, gamma, y=None, slope=0.0, on=0):
    h, dn, _ = _parts(dy, x, mean, rstd, y, slope, on)
    g = dn * gamma
    return rstd[:, None] * (g - _m(g) - h * _m(g * h)), (dn * h).sum(0), dn.sum(0)


def backward_size(dy, x, mean, rstd, gamma, y=None, slope=0.0, on=0):
    h, dn, H = _parts(dy, x, mean, rstd, y, slope, on)
    g, dn = (dn * gamma).abs(), dn.abs()
    return rstd[:, None] * (g + _m(g) + H * _m(g * H)), (dn * H).sum(0), dn.sum(0)


def backward2(u, dy, x, mean, rstd, gamma, y=None, slope=0.0, on=0):
    h, dn, _ = _parts(dy, x, mean, rstd, y, slope, on)
    g, r = dn * gamma, rstd[:, None]
    mg, mu, cg, cu = _m(g), _m(u), _m(g * h), _m(u * h)
    q = r * (u - mu - h * cu)
    ddy = gamma * q
    if on:
        ddy = torch.where(y > 0, ddy, slope * ddy)
    dx = r * r * (h * (3 * cg * cu + mg * mu - _m(g * u)) - cu * (g - mg) - cg * (u - mu))
    return ddy, dx, (dn * q).sum(0)


def backward2_size(u, dy, x, mean, rstd, gamma, y=None, slope=0.0, on=0):
    h, dn, H = _parts(dy, x, mean, rstd, y, slope, on)
    g, u, dn, r = (dn * gamma).abs(), u.abs(), dn.abs(), rstd[:, None]
    mg, mu, cg, cu = _m(g), _m(u), _m(g * H), _m(u * H)
    q = r * (u + mu + H * cu)
    return gamma.abs() * q, r * r * (H * (3 * cg * cu + mg * mu + _m(g * u)) + cu * (g + mg) + cg * (u + mu)), (dn * q).sum(0)


def orthogonalize(x, steps=5, coefficients=(3.4445, -4.7750, 2.0315), eps=1e-7):
    c = [coefficients] * steps if not hasattr(coefficients[0], '__len__') else list(coefficients)
    c = c * steps if len(c) == 1 else c
    if x.shape[0] < x.shape[1]:
        return orthogonalize(x.t(), steps, c, eps).t()
    norm = math.sqrt(float((x * x).sum())) + eps
    x = x / norm if norm > 0 else x
    for a, b, d in c:
        A = x.t() @ x
        x = a * x + x @ (b * A + d * (A @ A))
    return x


def muon(w, g, m, lr, momentum=0.95, nesterov=True, weight_decay=0.0, scale=None, **kw):
    m = momentum * m + g
    u = g + momentum * m if nesterov else m
    s = math.sqrt(max(1.0, w.shape[1] / w.shape[0])) if scale is None else scale
    return (1 - lr * weight_decay) * w - lr * s * orthogonalize(u, **kw), m
