"""Layer-normalised generators and critics and the Muon optimizer through the training functions, against float64 autograd.

Tolerances.  Every float32 result is a chain of at most some twenty products; each rounds its terms by 2^-24 relative to
them.  What relative errors of 2^-21 (eight such roundings) in every weight and input do to a result is computed for each
case, by running the float64 oracle on entries moved by +-2^-21: 16 of those responses, in the largest entry of the tensor,
are allowed, plus 16 roundings of the result itself (of its terms, where they cancel: the critic's output bias).  The seeds are such that no value in front of an activation is nearer
to zero than 4e-6 (asserted), so that no rounding flips a mask."""
import os
import socket
import sys

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

# G, hidden widths, batch, slope, layer norm in (generator, critic), seed
CASES = [
    (37, (16, 8), 5, 0.0, (True, True), 1),
    (37, (16,), 1, 0.0, (True, True), 1),
    (61, (24, 17, 5), 9, 0.2, (True, True), 1),
    (61, (24, 16), 33, 0.0, (True, False), 1),
    (61, (24, 16), 33, 0.1, (False, True), 2),
    (300, (13, 3), 6, 0.2, (True, True), 1),
    (700, (64, 48), 70, 0.0, (True, True), 1),
    (4297, (128, 128), 32, 0.0, (True, True), 1),
    (1077, (600, 130), 21, 0.0, (True, True), 2),
]


def case(G, H, B, slope, which, seed):
    """Problem of helpers.make_problem with layer-norm vectors: (dict of float32 arrays, generator, critic parameters)."""
    from helpers import make_problem
    from oracle import cgan_norm_oracle as N
    p = make_problem(G=G, V=(15, 3), H=H, Z=6, B=B, seed=seed, num_zero=False)
    for key, on, s in (('gp', which[0], 11), ('dp', which[1], 12)):
        if on:
            p[key]['ln'] = N.init_ln(H, seed + s)
    f = lambda a: np.asarray(a, np.float32)
    for key in ('gp', 'dp'):
        p[key] = N.rebuild(p[key], [f(a) for a in N.params(p[key])])
    for key in ('x', 'z', 'nc', 'alpha'):
        p[key] = f(p[key])
    return p


def tensors(q, rel=0.0, seed=0):
    """float64 copies of a problem's arrays, moved by +-rel."""
    from oracle import cgan_norm_oracle as N
    rs = np.random.RandomState(seed)
    mv = lambda a: torch.tensor(np.asarray(a, np.float64) * (1 + rel * rs.choice([-1.0, 1.0], size=np.shape(a))))
    out = {k: N.rebuild(q[k], [mv(a) for a in N.params(q[k])]) for k in ('gp', 'dp')}
    out.update({k: mv(q[k]) for k in ('x', 'z', 'nc', 'alpha')})
    out['cc'] = torch.tensor(q['cc'].astype(np.int64))
    return out


def oracle(t, slope):
    """[critic loss, its gradients..., generator loss, its gradients...]"""
    from oracle import cgan_norm_oracle as N
    dl, dg = N.disc_loss_and_grads(t['x'], t['z'], t['cc'], t['nc'], t['gp'], t['dp'], t['alpha'], slope=slope)
    gl, gg = N.gen_loss_and_grads(t['z'], t['cc'], t['nc'], t['gp'], t['dp'], slope=slope)
    return [dl.reshape(1)] + dg + [gl.reshape(1)] + gg


def margin(t, slope):
    """Smallest distance of a value in front of an activation from zero."""
    from oracle import cgan_norm_oracle as N
    seen = []
    with torch.no_grad():
        fake = N.forward(t['gp'], t['z'], t['cc'], t['nc'], slope=slope, seen=seen)
        for x in (t['x'], fake, t['x'] + t['alpha'] * (fake - t['x'])):
            N.forward(t['dp'], x, t['cc'], t['nc'], slope=slope, seen=seen)
    return min(float(s.abs().min()) for s in seen)


def params(q):
    from oracle import cgan_norm_oracle as N
    return N.params(q)


def allowed(q, slope):
    """(oracle results, allowed absolute errors)."""
    want = oracle(tensors(q), slope)
    tol = [16 * 2.0 ** -24 * float(w.abs().max()) for w in want]
    tol[len(want) - 2 - len(params(q['gp']))] += 16 * 2.0 ** -24 * 2     # the critic's output bias: 2B terms of +-1 / B
    moved = [oracle(tensors(q, 2.0 ** -21, s), slope) for s in (1, 2)]
    return want, [t + 16 * max(float((m[i] - want[i]).abs().max()) for m in moved) for i, t in enumerate(tol)]


def nets(T, p, slope):
    from oracle import cgan_norm_oracle as N
    ln = [bool(p[k].get('ln')) for k in ('gp', 'dp')]
    gen = T.Generator(p['G'], p['V'], p['n_num'], list(p['H']), p['Z'], slope=slope, weights=N.params(p['gp']), layer_norm=ln[0])
    disc = T.Critic(p['G'], p['V'], p['n_num'], list(p['H']), 1, slope=slope, weights=N.params(p['dp']), layer_norm=ln[1])
    return gen, disc


@pytest.mark.parametrize('G,H,B,slope,which,seed', CASES)
def test_gradients_of_both_steps(gpu, G, H, B, slope, which, seed):
    from adversarial_gene_expression_amd import tf_utils as T
    p = case(G, H, B, slope, which, seed)
    assert margin(tensors(p), slope) > 4e-6
    want, tol = allowed(p, slope)
    gen, disc = nets(T, p, slope)
    dl = T.train_disc(p['x'], p['z'], p['cc'], p['nc'], gen, disc, T.RMSprop(5e-4), alpha=p['alpha'], apply=False)
    gl = T.train_gen(p['z'], p['cc'], p['nc'], gen, disc, T.RMSprop(5e-4), apply=False)
    got = [np.float64(dl).reshape(1)] + disc.get_gradients() + [np.float64(gl).reshape(1)] + gen.get_gradients()
    assert len(got) == len(want)
    for i, (a, w, t) in enumerate(zip(got, want, tol)):
        err = float(np.abs(np.asarray(a, np.float64) - w.numpy().reshape(np.shape(a))).max())
        assert err <= t, (i, np.shape(a), err, t)


@pytest.mark.parametrize('G,H,B,slope,which,seed', CASES[:3])
def test_gradients_against_differences(gpu, G, H, B, slope, which, seed):
    """The gradient's product with a random direction against the central difference of the float64 loss along it: h = 1e-6
    leaves h^2 times a third derivative and 2^-53 / h, both far below the gradient's own allowance."""
    from adversarial_gene_expression_amd import tf_utils as T
    from oracle import cgan_norm_oracle as N
    p = case(G, H, B, slope, which, seed)
    gen, disc = nets(T, p, slope)
    T.train_disc(p['x'], p['z'], p['cc'], p['nc'], gen, disc, T.RMSprop(5e-4), alpha=p['alpha'], apply=False)
    T.train_gen(p['z'], p['cc'], p['nc'], gen, disc, T.RMSprop(5e-4), apply=False)
    _, tol = allowed(p, slope)
    t = tensors(p)
    nd = len(N.params(p['dp']))
    for net, key, tols in ((disc, 'dp', tol[1:1 + nd]), (gen, 'gp', tol[2 + nd:])):
        rs = np.random.RandomState(7)
        v = [torch.tensor(rs.randn(*np.shape(a))) for a in N.params(p[key])]

        def loss(h):
            q = dict(t, **{key: N.rebuild(t[key], [a + h * b for a, b in zip(N.params(t[key]), v)])})
            if key == 'dp':
                return float(N.disc_loss(q['x'], q['z'], q['cc'], q['nc'], q['gp'], q['dp'], q['alpha'], slope=slope).detach())
            return float(N.gen_loss(q['z'], q['cc'], q['nc'], q['gp'], q['dp'], slope=slope))
        h = 1e-6
        want = (loss(h) - loss(-h)) / (2 * h)
        got = sum(float((torch.tensor(g, dtype=torch.float64).reshape(b.shape) * b).sum()) for g, b in zip(net.get_gradients(), v))
        room = sum(a * float(b.abs().sum()) for a, b in zip(tols, v)) + 1e-7 * max(1.0, abs(want))
        assert abs(got - want) <= room, (key, got, want, room)


def test_augmented_critic_step(gpu):
    from adversarial_gene_expression_amd import tf_utils as T
    from oracle import cgan_norm_oracle as N
    p = case(61, (24, 16), 9, 0.0, (True, True), 4)
    rs = np.random.RandomState(2)
    aug = dict(mask=np.asarray(rs.binomial(1, 0.5, 9), np.float32), noise_fake=np.asarray(0.5 * rs.randn(61), np.float32),
               noise_real=np.asarray(0.5 * rs.randn(9, 61), np.float32))
    gen, disc = nets(T, p, 0.0)
    loss = T.train_disc(p['x'], p['z'], p['cc'], p['nc'], gen, disc, T.RMSprop(5e-4), alpha=p['alpha'], aug=aug, apply=False)
    # the same without augmentation on rows that hold it already: the fake rows by the generator's output bias (one row
    # of noise for all of them, so a mask of ones), the real rows as given
    p2 = dict(p, x=p['x'] + aug['mask'][:, None] * aug['noise_real'])
    ones = dict(aug, mask=np.ones(9, np.float32), noise_real=np.zeros((9, 61), np.float32))
    l1 = T.train_disc(p2['x'], p['z'], p['cc'], p['nc'], gen, disc, T.RMSprop(5e-4), alpha=p['alpha'], aug=ones, apply=False)
    t = tensors(p2)
    t['gp']['b'][-1] = t['gp']['b'][-1] + torch.tensor(aug['noise_fake'].astype(np.float64))
    want, grads = N.disc_loss_and_grads(t['x'], t['z'], t['cc'], t['nc'], t['gp'], t['dp'], t['alpha'])
    q = dict(p2, gp=N.rebuild(p2['gp'], [a.numpy() for a in N.params(t['gp'])]))
    _, tol = allowed(q, 0.0)
    assert np.isfinite(float(loss)) and abs(float(l1) - float(want)) <= tol[0]
    for a, w, b in zip(disc.get_gradients(), grads, tol[1:]):
        assert float(np.abs(a - w.numpy().reshape(a.shape)).max()) <= b


@pytest.mark.parametrize('G,H,B,slope,which,seed', CASES[:4])
def test_models_forward_penalty_and_files(gpu, tmp_path, G, H, B, slope, which, seed):
    from adversarial_gene_expression_amd import tf_utils as T
    from oracle import cgan_norm_oracle as N, cgan_oracle as O
    p = case(G, H, B, slope, which, seed)
    gen, disc = nets(T, p, slope)
    t, m = tensors(p), tensors(p, 2.0 ** -21, 3)

    def results(t):
        fake = N.forward(t['gp'], t['z'], t['cc'], t['nc'], slope=slope)
        return (fake, N.forward(t['dp'], t['x'], t['cc'], t['nc'], slope=slope),
                O.gradient_penalty(lambda x: N.forward(t['dp'], x, t['cc'], t['nc'], slope=slope), t['x'], fake.detach(),
                                   t['alpha']).reshape(1))
    want, moved = results(t), results(m)
    fake = T.predict(p['cc'], p['nc'], gen, z=p['z'])
    got = (fake, np.asarray(disc([p['x'], p['cc'], p['nc']])),
           np.asarray(T.gradient_penalty(lambda x: disc([x, p['cc'], p['nc']], training=True), p['x'], fake, alpha=p['alpha'])))
    for a, w, v in zip(got, want, moved):
        w = w.detach().numpy().reshape(np.shape(a))
        tol = 16 * float(np.abs(v.detach().numpy().reshape(np.shape(a)) - w).max()) + 2.0 ** -20 * float(np.abs(w).max())
        assert float(np.abs(a - w).max()) <= tol
    for k, net in enumerate((gen, disc)):
        path = str(tmp_path / ('net%d' % k))
        net.save(path)
        again = T.load_model(path)
        assert again.layer_norm == which[k] and again.ln_epsilon == net.ln_epsilon
        for a, b in zip(net.get_weights(), again.get_weights()):
            np.testing.assert_array_equal(a, b)
    names = len(gen.trainable_variables)
    assert names == len(gen.get_weights()) == 2 + 2 * (len(H) + 1) + (2 * len(H) if which[0] else 0)


def is_kernel(ws, i):
    """A Dense kernel with both sides above 1: a matrix in front of a vector of its column count."""
    return ws[i].ndim == 2 and min(ws[i].shape) > 1 and ws[i + 1].shape == ws[i].shape[1:]


def muon_step(ws, grads, m, rms, opt, fb):
    """What one step should leave: (weights, allowed error per tensor, momentum, fallback slots), by the float64 formulas."""
    from test_gpu_orth import allowed as orth_allowed
    out, tols, ms, slots = [], [], [], []
    for i, (w, g, a, r) in enumerate(zip(ws, grads, m, rms)):
        w, g = np.asarray(w, np.float64), np.asarray(g, np.float64)
        if is_kernel(ws, i):
            a = opt.momentum * a + g
            o, tol = orth_allowed(torch.tensor(g + opt.momentum * a if opt.nesterov else a))
            s = opt.learning_rate * max(1.0, w.shape[1] / w.shape[0]) ** 0.5
            out.append((1 - opt.learning_rate * opt.weight_decay) * w - s * o.numpy())
            tols.append(s * tol * float(np.linalg.norm(o.numpy())) + 2.0 ** -22 * np.abs(w).max())
        else:
            r = fb.rho * r + (1 - fb.rho) * g * g
            out.append(w - fb.learning_rate * g / (np.sqrt(r) + fb.epsilon))
            tols.append(2.0 ** -22 * np.abs(w).max() + 2.0 ** -19 * fb.learning_rate * 10 ** 0.5)
        ms.append(a)
        slots.append(r)
    return out, tols, ms, slots


@pytest.mark.parametrize('ln', [True, False])
@pytest.mark.parametrize('kw', [dict(), dict(nesterov=False, momentum=0.9, weight_decay=0.1)])
def test_muon_steps_of_both_nets(gpu, ln, kw):
    """Three steps of each net; every step from the product's own weights, momentum and gradients of that moment (float32),
    so that one step's rounding is judged at a time."""
    from adversarial_gene_expression_amd import tf_utils as T
    p = case(130, (24, 16), 20, 0.0, (ln, ln), 2)
    gen, disc = nets(T, p, 0.0)
    for net, other in ((disc, gen), (gen, disc)):
        opt = T.tfk.optimizers.Muon(0.02, fallback=T.RMSprop(1e-3), **kw)
        shapes = [w.shape for w in net.get_weights()]
        m, r = [np.zeros(s) for s in shapes], [np.zeros(s) for s in shapes]
        for step in range(3):
            z = np.random.RandomState(step).randn(20, 6).astype(np.float32)
            if net is disc:
                T.train_disc(p['x'], z, p['cc'], p['nc'], gen, disc, opt, alpha=p['alpha'], apply=False)
            else:
                T.train_gen(z, p['cc'], p['nc'], gen, disc, opt, apply=False)
            before, g = net.get_weights(), net.get_gradients()
            opt.apply(net)
            want, tol, m, r = muon_step(before, g, m, r, opt, opt.fallback)
            state = opt.state_arrays(net)
            for i, (a, w, t) in enumerate(zip(net.get_weights(), want, tol)):
                assert float(np.abs(a - w).max()) <= t, (step, i, a.shape, float(np.abs(a - w).max()), t)
            for i, (a, v, mm, rms, rr) in enumerate(zip(before, state['momentum'], m, state['rms'], r)):
                on = is_kernel(before, i)
                np.testing.assert_allclose(v, mm if on else np.zeros_like(a), rtol=0, atol=2.0 ** -21 * np.abs(mm).max() if on else 0)
                np.testing.assert_allclose(rms, rr if not on else np.zeros_like(a), rtol=2.0 ** -20, atol=0)
            m, r = [np.asarray(v, np.float64) for v in state['momentum']], [np.asarray(v, np.float64) for v in state['rms']]
        assert opt.iterations == 3 and opt.fallback.iterations == 3


def test_train_runs_normalised_nets_with_muon(gpu):
    """train() on a ragged last batch = the step functions in its order, bit for bit; the captured iteration refuses both."""
    from adversarial_gene_expression_amd import _lib, tf_utils as T
    p = case(61, (24, 16), 23, 0.0, (True, True), 4)
    ws = []
    for manual in (False, True):
        gen, disc = nets(T, p, 0.0)
        go, do = T.Muon(0.01), T.Muon(0.01, fallback=T.Adam(1e-3))
        T.set_seed(5)
        if not manual:
            tr = T.train(p['x'], p['cc'], p['nc'], 6, 2, 10, gen, disc, lambda g: 0.0, lambda: None, gen_opt=go, disc_opt=do,
                         verbose=False, nb_critic=2)
            assert np.all(np.isfinite(tr['gen_loss'])) and np.all(np.isfinite(tr['disc_loss']))
            assert go.iterations == 6 and do.iterations == 12
        else:
            for _ in range(2):
                for lo, hi in ((0, 10), (10, 20), (20, 23)):
                    x, cc, nc = p['x'][lo:hi], p['cc'][lo:hi], p['nc'][lo:hi]
                    for _ in range(2):
                        z, al = T.random_normal((hi - lo, 6)), T.random_uniform((hi - lo, 1))
                        T.train_disc(x, z, cc, nc, gen, disc, do, alpha=al)
                    T.train_gen(T.random_normal((hi - lo, 6)), cc, nc, gen, disc, go)
        ws.append(gen.get_weights() + disc.get_weights())
        assert all(np.all(np.isfinite(w)) for w in ws[-1])
    for a, b in zip(*ws):
        np.testing.assert_array_equal(a, b)
    with pytest.raises(ValueError):
        T.train_iteration(p['x'], p['cc'], p['nc'], gen, disc, T.RMSprop(5e-4), T.RMSprop(5e-4))
    with pytest.raises(_lib.AgxError):
        T._pair(gen, disc, 23).iteration_graph(gen, disc, T.RMSprop(5e-4), T.RMSprop(5e-4), 23, 2, 10.0, 1)


def test_one_set_of_buffers_serves_smaller_batches_and_other_streams(gpu):
    """The step's buffers are made for the largest batch: a smaller one behind it, and the same on another stream, give what
    fresh nets give."""
    from adversarial_gene_expression_amd import tf_utils as T
    p = case(61, (24, 16), 33, 0.0, (True, True), 1)
    gen, disc = nets(T, p, 0.0)

    def grads(gen, disc, n):
        T.train_disc(p['x'][:n], p['z'][:n], p['cc'][:n], p['nc'][:n], gen, disc, T.RMSprop(5e-4), alpha=p['alpha'][:n], apply=False)
        T.train_gen(p['z'][:n], p['cc'][:n], p['nc'][:n], gen, disc, T.RMSprop(5e-4), apply=False)
        return disc.get_gradients() + gen.get_gradients()
    big = grads(gen, disc, 33)
    for n in (1, 4, 33):
        fresh = grads(*nets(T, p, 0.0), n)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            other = grads(gen, disc, n)
        torch.cuda.current_stream().wait_stream(s)
        for a, b in zip(other, fresh):
            np.testing.assert_array_equal(a, b)
    for a, b in zip(big, fresh):
        np.testing.assert_array_equal(a, b)


def _run(out_path):
    sys.path.insert(0, os.path.join(ROOT, 'tests'))
    from adversarial_gene_expression_amd import tf_utils as T
    p = case(61, (24, 16), 23, 0.0, (True, True), 4)
    gen, disc = nets(T, p, 0.0)
    world, rank = T._world()
    lo, hi = T._shard(0, 23, world, rank)
    s = slice(lo, hi)
    do, go = T.Muon(0.01), T.Muon(0.01, fallback=T.Adam(1e-3))
    dl = T.train_disc(p['x'][s], p['z'][s], p['cc'][s], p['nc'][s], gen, disc, do, alpha=p['alpha'][s], batch_global=23)
    gl = T.train_gen(p['z'][s], p['cc'][s], p['nc'][s], gen, disc, go, batch_global=23)
    st = do.state_arrays(disc)
    out = dict(dl=np.float64(dl), gl=np.float64(gl))
    for k, ws in (('d', disc.get_weights()), ('g', gen.get_weights()), ('m', st['momentum']), ('r', st['rms']),
                  ('v', go.state_arrays(gen)['v'])):
        out.update({'%s%02d' % (k, i): w for i, w in enumerate(ws)})
    np.savez(out_path, **out)


def _worker(rank, world, port, out_dir):
    os.environ.update(MASTER_ADDR='127.0.0.1', MASTER_PORT=str(port))
    import torch.distributed as dist
    dist.init_process_group('gloo', rank=rank, world_size=world)
    try:
        _run(os.path.join(out_dir, 'rank%d.npz' % rank))
    finally:
        dist.destroy_process_group()


def test_two_ranks_take_the_one_process_step(gpu, tmp_path):
    """Two data-parallel ranks hold the same bits, and the weights of the one-process run of the whole batch: the ranks'
    gradients differ from its own in the order of their sums only, so the tolerance is the response of the float64 step to
    gradients off by the allowance of test_gradients_of_both_steps."""
    import torch.multiprocessing as mp
    from adversarial_gene_expression_amd import tf_utils as T
    from oracle import norm_oracle as N
    with socket.socket() as s:
        s.bind(('127.0.0.1', 0))
        port = s.getsockname()[1]
    _run(str(tmp_path / 'ref.npz'))
    mp.spawn(_worker, args=(2, port, str(tmp_path)), nprocs=2, join=True)
    ref, r0, r1 = (np.load(str(tmp_path / n)) for n in ('ref.npz', 'rank0.npz', 'rank1.npz'))
    for k in ref.files:
        np.testing.assert_array_equal(r0[k], r1[k])
    p = case(61, (24, 16), 23, 0.0, (True, True), 4)
    want, tol = allowed(p, 0.0)
    assert abs(float(r0['dl']) - float(ref['dl'])) <= 2 * tol[0]
    # the critic's kernels after one step from zero momentum: u = (1 + momentum) g, and its orthogonalised form responds to
    # an error e of g as the oracle's does
    _, disc = nets(T, p, 0.0)
    ws = disc.get_weights()
    rs = np.random.RandomState(0)
    for i, (w, g, t) in enumerate(zip(ws, want[1:], tol[1:])):
        diff = float(np.abs(r0['d%02d' % i] - ref['d%02d' % i]).max())
        if is_kernel(ws, i):
            e = torch.tensor(rs.uniform(-t, t, size=w.shape))
            s = 0.01 * max(1.0, w.shape[1] / w.shape[0]) ** 0.5
            o = N.orthogonalize(g)
            resp = float((N.orthogonalize(g + e) - o).abs().max())
            assert diff <= s * (4 * resp + 2.0 ** -18), (i, diff, resp)
        else:
            assert diff <= 2 * 5e-4 * 10 ** 0.5     # (the first RMSprop step is lr sqrt(10) sign(g): a flipped sign of g ~ 0)
        np.testing.assert_allclose(r0['m%02d' % i], ref['m%02d' % i], rtol=0, atol=4 * t)


def test_whatever_memory_held_before_stays_out(gpu):
    """Odd widths leave padding behind the rows of intermediate results: memory full of NaN changes nothing."""
    from adversarial_gene_expression_amd import tf_utils as T
    p = case(61, (24, 17, 5), 9, 0.2, (True, True), 1)
    gen, disc = nets(T, p, 0.2)

    def run():
        junk = [torch.full((n,), float('nan'), device=gpu) for n in [64, 192, 256, 512, 1024, 4096, 1 << 16, 1 << 20] * 8]
        del junk
        fake = T.predict(p['cc'], p['nc'], gen, z=p['z'])
        return (fake, np.asarray(disc([p['x'], p['cc'], p['nc']])),
                np.asarray(T.gradient_penalty(lambda x: disc([x, p['cc'], p['nc']], training=True), p['x'], fake, alpha=p['alpha'])))
    first = run()
    for a, b in zip(first, run()):
        assert np.all(np.isfinite(a))
        np.testing.assert_array_equal(a, b)


def test_c_forward_entries(gpu):
    """agx_cgan_gen_forward / disc_forward of normalised nets, the critic over up to three times the batch, against __call__."""
    from adversarial_gene_expression_amd import _dev, _lib, tf_utils as T
    p = case(61, (24, 17, 5), 33, 0.2, (True, True), 1)
    gen, disc = nets(T, p, 0.2)
    pair, lib = T._pair(gen, disc, 33), _lib.load()
    x, z, nc = (_dev.to_dev(p[k]) for k in ('x', 'z', 'nc'))
    cc = _dev.to_dev(p['cc'], torch.int32)
    out = torch.empty(33, 61, device=gpu)
    _lib.check(lib.agx_cgan_gen_forward(pair.handle, _dev.stream(), z.data_ptr(), cc.data_ptr(), nc.data_ptr(), 33, out.data_ptr(), 61))
    want = torch.as_tensor(np.asarray(gen([z, cc, nc])), device=gpu)
    assert float((out - want).abs().max()) <= 2.0 ** -18 * float(want.abs().max())
    x3, cc3, nc3 = (t.repeat(3, 1).contiguous() for t in (x, cc, nc))
    rows = 3 * pair.max_batch if 3 * pair.max_batch <= 99 else 99
    s = torch.empty(rows, device=gpu)
    _lib.check(lib.agx_cgan_disc_forward(pair.handle, _dev.stream(), x3.data_ptr(), 61, cc3.data_ptr(), nc3.data_ptr(), rows, s.data_ptr()))
    want = torch.as_tensor(np.asarray(disc([x3[:rows], cc3[:rows], nc3[:rows]])), device=gpu).reshape(-1)
    assert float((s - want).abs().max()) <= 2.0 ** -18 * float(want.abs().max())


@pytest.mark.parametrize('G,H,B,slope,which,seed', [CASES[2], CASES[3], CASES[4]])
def test_augmented_steps_of_both_nets(gpu, G, H, B, slope, which, seed):
    """Losses and gradients with noise on some of the rows (one row of it for all fake ones, tf_utils.py:209; a row each for
    the generator's, :247), against the float64 oracle on the augmented rows; the noise is moved as the inputs are."""
    from adversarial_gene_expression_amd import tf_utils as T
    from oracle import cgan_norm_oracle as N, cgan_oracle as O
    p = case(G, H, B, slope, which, seed)
    rs = np.random.RandomState(seed + 40)
    f = lambda *s: np.asarray(0.5 * rs.randn(*s), np.float32)  # noqa: E731
    mask = np.asarray(np.arange(B) % 3 != 1, np.float32)
    noise = dict(fake=f(G), real=f(B, G), gen=f(B, G))
    m = torch.tensor(mask.astype(np.float64))[:, None]

    def both(t, e, seen=None):
        net = lambda key, x, **kw: N.forward(t[key], x, t['cc'], t['nc'], slope=slope, seen=seen, **kw)  # noqa: E731
        ps = [a.detach().requires_grad_(True) for a in N.params(t['dp'])]
        q = dict(t, dp=N.rebuild(t['dp'], ps))
        with torch.no_grad():
            fake = net('gp', t['z']) + m * e['fake']
        real = t['x'] + m * e['real']
        critic = lambda x: N.forward(q['dp'], x, t['cc'], t['nc'], slope=slope, seen=seen)  # noqa: E731
        loss = O.discriminator_loss(critic(real), critic(fake)) + 10.0 * O.gradient_penalty(critic, real, fake, t['alpha'])
        out = [loss.detach().reshape(1)] + N._grads(loss, ps)
        ps = [a.detach().requires_grad_(True) for a in N.params(t['gp'])]
        made = N.forward(N.rebuild(t['gp'], ps), t['z'], t['cc'], t['nc'], slope=slope, seen=seen) + m * e['gen']
        loss = O.generator_loss(net('dp', made))
        return out + [loss.detach().reshape(1)] + N._grads(loss, ps)

    def moved(rel, s):
        r = np.random.RandomState(s + 90)
        return both(tensors(p, rel, s), {k: torch.tensor(v.astype(np.float64) * (1 + rel * r.choice([-1.0, 1.0], size=v.shape)))
                                         for k, v in noise.items()}, seen)
    seen = []
    want = moved(0.0, 0)
    assert min(float(v.abs().min()) for v in seen) > 4e-6
    tol = [16 * 2.0 ** -24 * float(w.abs().max()) for w in want]
    tol[len(params(p['dp']))] += 16 * 2.0 ** -24 * 2          # the critic's output bias, as in allowed()
    others = [moved(2.0 ** -21, s) for s in (1, 2)]
    tol = [t + 16 * max(float((o[i] - want[i]).abs().max()) for o in others) for i, t in enumerate(tol)]
    gen, disc = nets(T, p, slope)
    dl = T.train_disc(p['x'], p['z'], p['cc'], p['nc'], gen, disc, T.RMSprop(5e-4), alpha=p['alpha'], apply=False,
                      aug=dict(mask=mask, noise_fake=noise['fake'], noise_real=noise['real']))
    gl = T.train_gen(p['z'], p['cc'], p['nc'], gen, disc, T.RMSprop(5e-4), apply=False, aug=dict(mask=mask, noise=noise['gen']))
    got = [np.float64(dl).reshape(1)] + disc.get_gradients() + [np.float64(gl).reshape(1)] + gen.get_gradients()
    assert len(got) == len(want)
    for i, (a, w, t) in enumerate(zip(got, want, tol)):
        err = float(np.abs(np.asarray(a, np.float64) - w.numpy().reshape(np.shape(a))).max())
        assert err <= t, (i, np.shape(a), err, t)
