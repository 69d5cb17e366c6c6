"""Torch-CPU autograd oracle of the optional layer-normalised generator and critic.

TEST INFRASTRUCTURE ONLY (see ``oracle/__init__.py``).  NO REFERENCE COUNTERPART: the reference's nets are Dense + ReLU
(``tf_utils.py:85-88``, ``:132-135``), so this pins nothing against the reference.  It restates Keras
``LayerNormalization()`` (epsilon 1e-3, biased variance, gamma 1 / beta 0) behind every hidden Dense and in front of the
activation; parameters are those of ``cgan_oracle`` with an optional entry ``ln``: [(gamma, beta)] per hidden layer.
"""
import numpy as np
import torch

from . import cgan_oracle as O


def init_ln(h_dims, seed):
    rs = np.random.RandomState(seed)
    return [(rs.uniform(0.5, 1.5, n), rs.uniform(-0.3, 0.3, n)) for n in h_dims]


def params(p):
    """Keras variable order: embeddings, then per layer kernel, bias (, gamma, beta)."""
    out = list(p['emb'])
    for i, (w, b) in enumerate(zip(p['W'], p['b'])):
        out += [w, b]
        if p.get('ln') and i < len(p['ln']):
            out += list(p['ln'][i])
    return out


def rebuild(p, tensors):
    """The same structure with other tensors, given in the order of params()."""
    it = iter(tensors)
    q = {'emb': [next(it) for _ in p['emb']], 'W': [], 'b': []}
    if p.get('ln'):
        q['ln'] = []
    for i in range(len(p['W'])):
        q['W'].append(next(it))
        q['b'].append(next(it))
        if p.get('ln') and i < len(p['ln']):
            q['ln'].append((next(it), next(it)))
    return q


def mlp(p, h, slope=0.0, eps=1e-3, seen=None):
    """seen: a list that takes the values in front of every activation."""
    n = len(p['W'])
    for i in range(n):
        h = h @ p['W'][i] + p['b'][i]
        if i < n - 1:
            if p.get('ln'):
                gamma, beta = p['ln'][i]
                mu = h.mean(1, keepdim=True)
                h = gamma * (h - mu) / torch.sqrt(((h - mu) ** 2).mean(1, keepdim=True) + eps) + beta
            if seen is not None:
                seen.append(h.detach())
            h = torch.where(h > 0, h, slope * h)
    return h


def forward(p, lead, cc, nc, **kw):
    return mlp(p, torch.cat([lead, O._cov_features(p, cc, nc)], dim=-1), **kw)


def _grads(loss, ps):
    got = torch.autograd.grad(loss, ps, allow_unused=True)
    return [torch.zeros_like(p) if g is None else g for g, p in zip(got, ps)]


def disc_loss(x, z, cc, nc, gen_p, disc_p, alpha, weight=10.0, **kw):
    with torch.no_grad():
        fake = forward(gen_p, z, cc, nc, **kw)
    gp = O.gradient_penalty(lambda xi: forward(disc_p, xi, cc, nc, **kw), x, fake, alpha)
    return O.discriminator_loss(forward(disc_p, x, cc, nc, **kw), forward(disc_p, fake, cc, nc, **kw)) + weight * gp


def gen_loss(z, cc, nc, gen_p, disc_p, **kw):
    return O.generator_loss(forward(disc_p, forward(gen_p, z, cc, nc, **kw), cc, nc, **kw))


def disc_loss_and_grads(x, z, cc, nc, gen_p, disc_p, alpha, **kw):
    """tf_utils.py:186-220."""
    ps = [t.detach().requires_grad_(True) for t in params(disc_p)]
    loss = disc_loss(x, z, cc, nc, gen_p, rebuild(disc_p, ps), alpha, **kw)
    return loss.detach(), _grads(loss, ps)


def gen_loss_and_grads(z, cc, nc, gen_p, disc_p, **kw):
    """tf_utils.py:226-255."""
    ps = [t.detach().requires_grad_(True) for t in params(gen_p)]
    loss = gen_loss(z, cc, nc, rebuild(gen_p, ps), disc_p, **kw)
    return loss.detach(), _grads(loss, ps)
