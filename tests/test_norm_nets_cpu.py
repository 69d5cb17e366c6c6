"""Layer-normalised nets and Muon: layouts and refusals that need no GPU."""
from types import SimpleNamespace

import pytest

from adversarial_gene_expression_amd import _lib, tf_utils as T


def test_normalisations_exclude_each_other():
    for cls in (T.Generator, T.Critic):
        with pytest.raises((ValueError, NotImplementedError)):
            cls(37, [15, 3], 1, [16, 8], 6, batch_norm=True, layer_norm=True)
        for eps in (0.0, -1.0, float('nan')):
            with pytest.raises(ValueError):
                cls(37, [15, 3], 1, [16, 8], 6, layer_norm=True, ln_epsilon=eps)


def test_model_files_with_malformed_layer_norm_entries():
    good = dict(kind='disc', x_dim=5, z_dim=1, nb_numeric=1, vocab_sizes=[3], h_dims=[4], slope=0.0, layer_norm=True, ln_epsilon=1e-3)
    assert T._check_model_config(good)['layer_norm'] is True
    assert 'layer_norm' not in T._check_model_config({k: v for k, v in good.items() if not k.startswith('l')})
    for bad in (dict(layer_norm=2), dict(ln_epsilon=0.0), dict(ln_epsilon='1'), dict(ln_epsilon=None),
                dict(batch_norm=True, bn_epsilon=1e-3, bn_momentum=0.9)):
        with pytest.raises(ValueError):
            T._check_model_config(dict(good, **bad))


def _net(x_dim, h, kind, **kw):
    """The flat layout of a net, without its device buffers."""
    cls = T.Generator if kind == 'gen' else T.Critic
    net = cls.__new__(cls)
    net.batch_norm, net.layer_norm = False, kw.get('layer_norm', False)
    net.bn_epsilon, net.bn_momentum, net.ln_epsilon = 1e-3, 0.99, 1e-3
    net.vocab_sizes, net.emb_dims, net.nb_numeric = [15, 3], T._emb_dims([15, 3]), 1
    lead, out = (6, x_dim) if kind == 'gen' else (x_dim, 1)
    net.dims = [lead + 1 + sum(net.emb_dims)] + list(h) + [out]
    net._layout()
    return net


@pytest.mark.parametrize('kind', ['gen', 'disc'])
@pytest.mark.parametrize('ln', [False, True])
@pytest.mark.parametrize('h', [[16, 8], [7], [5, 1, 33]])
def test_muon_covers_every_parameter_once(kind, ln, h):
    net = _net(61, h, kind, layer_norm=ln)
    mats, gaps = T.Muon._plan(net)
    hit = [0] * net.n_flat
    for o, r, c, ld in mats:
        assert min(r, c) > 1 and o % 4 == 0
        for i in range(o, o + r * ld):
            hit[i] += 1
    for o, n in gaps:
        assert o % 4 == 0
        for i in range(o, o + n):
            hit[i] += 2
    for o, r, c, ld in net._segments():
        kernel = (o, r, c, ld) in mats
        assert all(hit[i] == (1 if kernel else 2) for i in range(o, o + r * ld))
    assert max(hit) <= 2
    want = sum(1 for a, b in zip(net.dims, net.dims[1:]) if min(a, b) > 1)
    assert len(mats) == want
    names = [s for s in net._segments()]
    assert len(names) == 2 + 2 * (len(h) + 1) + (2 * len(h) if ln else 0)


def test_muon_leaves_kernels_beyond_the_largest_side_to_the_fallback():
    big = _lib.AGX_ORTH_MAX_SIDE + 1
    net = SimpleNamespace(w_off=[0, 64], dims=[big, big, 4], ldw=[big + 3, 4], n_flat=64 + 4 * big + 192)
    mats, gaps = T.Muon._plan(net)
    assert mats == [(64, big, 4, 4)] and gaps[0] == (0, 64)


def test_muon_takes_rmsprop_or_adam_as_its_fallback():
    assert type(T.Muon().fallback) is T.RMSprop and T.tfk.optimizers.Muon is T.Muon
    assert T.Muon(lr=0.5).learning_rate == 0.5
    for bad in (T.Muon(), 'adam', 1e-3):
        with pytest.raises(TypeError):
            T.Muon(fallback=bad)
    for o in (T.Muon(), T.RMSprop()):
        assert not T._graph_ok(T.Muon(), o)


def _config():
    cfg = _lib.CganConfig()
    gen, disc = _net(37, [16, 8], 'gen', layer_norm=True), _net(37, [16, 8], 'disc', layer_norm=True)
    cfg.x_dim, cfg.z_dim, cfg.max_batch, cfg.max_steps = 37, 6, 32, 6
    cfg.gen, cfg.disc = gen.desc, disc.desc
    return cfg


def test_descriptors_of_normalised_nets():
    lib = _lib.load()

    def create(cfg):
        h = _lib.C.c_void_p()
        rc = lib.agx_cgan_create(cfg, _lib.C.byref(h))
        n = int(lib.agx_cgan_workspace_bytes(h)) if rc == 0 else 0
        if rc == 0:
            lib.agx_cgan_destroy(h)
        return rc, n
    rc, n = create(_config())
    assert rc == 0
    plain = _config()
    plain.gen.ln = plain.disc.ln = 0
    assert 0 < create(plain)[1] < n
    for bad in ('bn', 'eps', 'gamma', 'beta', 'odd'):
        cfg = _config()
        for m in (cfg.gen, cfg.disc):
            if bad == 'bn':
                m.bn, m.bn_eps, m.bn_momentum = 1, 1e-3, 0.9
            elif bad == 'eps':
                m.ln_eps = 0.0
            elif bad == 'gamma':
                m.ln_gamma_off[1] = m.n_flat
            elif bad == 'beta':
                m.ln_beta_off[0] = -4
            else:
                m.ln_beta_off[0] += 1
        assert create(cfg)[0] == -1, bad
