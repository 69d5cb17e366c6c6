"""Orthogonalised updates without a GPU: refusals, workspace queries, the oracle against the singular value decomposition."""
import pytest
import torch

from adversarial_gene_expression_amd import AgxError, _lib, ops
from oracle import norm_oracle as N


@pytest.mark.parametrize('x', [torch.zeros(8), torch.zeros(4, 8, dtype=torch.float64), torch.zeros(4, 0), torch.zeros(8, 4).t(),
                               torch.zeros(1, 8).expand(4, 8)])
def test_refuses_operands(x):
    with pytest.raises(ValueError):
        ops.orthogonalize(x)
    with pytest.raises(ValueError):
        ops.orthogonalize([torch.zeros(4, 4), x])
    with pytest.raises(ValueError):
        ops.muon(x, x, x, 0.1)


def test_refuses_arguments():
    x = torch.zeros(4, 6)
    for kw in (dict(steps=0), dict(steps=17), dict(steps=2.5), dict(coefficients=(1.0, 2.0)),
               dict(steps=3, coefficients=[(1.0, 0.0, 0.0)] * 2)):
        with pytest.raises(ValueError):
            ops.orthogonalize(x, **kw)
        with pytest.raises(ValueError):
            ops.muon(x, x.clone(), x.clone(), 0.1, **kw)
    b = x.to(torch.bfloat16)
    for w, g, m in ((b, b, b), (x, b, x), (x, torch.zeros(6, 4), x), ([x, x], [x], [x])):
        with pytest.raises(ValueError):
            ops.muon(w, g, m, 0.1)


def test_no_gpu_is_an_error():
    if torch.cuda.is_available():
        pytest.skip('GPU present')
    with pytest.raises(AgxError):
        ops.orthogonalize(torch.zeros(4, 6))
    with pytest.raises(AgxError):
        ops.muon(torch.zeros(4, 6), torch.zeros(4, 6), torch.zeros(4, 6), 0.1)


def _job(rows=4, cols=6, dtype=0):
    j = (_lib.OrthDesc * 1)()
    j[0].x, j[0].out, j[0].ldx, j[0].ldo, j[0].rows, j[0].cols, j[0].dtype = 4096, 8192, cols, cols, rows, cols, dtype
    return j


def _opts(steps=5, coef=(3.4445, -4.7750, 2.0315), eps=1e-7):
    o = _lib.OrthOpts()
    o.steps, o.n_coef, o.eps = steps, 1, eps
    for k, v in enumerate(coef):
        o.coef[k] = v
    return o


def test_abi_refuses_before_any_launch():
    lib = _lib.load()
    err = lambda: lib.agx_last_error().decode()  # noqa: E731
    big = 1 << 40
    run = lambda j, o, n=1, ws=4096, size=big: lib.agx_orthogonalize(None, j, n, o, ws, size)  # noqa: E731
    assert run(None, _opts()) == -1 and run(_job(), None) == -1 and run(_job(), _opts(), n=0) == -1 and run(_job(), _opts(), n=17) == -1
    assert run(_job(rows=0), _opts()) == -1 and run(_job(rows=4097, cols=5000), _opts()) == -1 and run(_job(dtype=2), _opts()) == -1
    for o in (_opts(steps=0), _opts(steps=17), _opts(eps=-1.0), _opts(eps=float('inf')), _opts(coef=(float('nan'), 0, 0))):
        assert run(_job(), o) == -1
    assert run(_job(), _opts(coef=(100.0, 0.0, 0.0))) == -1 and 'singular values' in err()   # diverges within five steps
    assert run(_job(), _opts(coef=(0.0, 0.0, 0.0))) == -1                                    # vanishes
    j = _job()
    j[0].ldx = 5
    assert run(j, _opts()) == -1
    j = _job()
    j[0].x = 4097
    assert run(j, _opts()) == -1 and 'aligned' in err()
    j = _job()
    j[0].out = j[0].x
    assert run(j, _opts()) == -1 and 'over the input' in err()
    assert run(_job(), _opts(), ws=None) == -3 and run(_job(), _opts(), size=16) == -3
    assert run(_job(), _opts(), ws=4100) == -1
    m = (_lib.MuonDesc * 1)()
    m[0].rows, m[0].cols, m[0].scale, m[0].ldw, m[0].ldg, m[0].ldm = 4, 6, 1.0, 6, 6, 6
    o = _lib.MuonOpts()
    o.orth, o.lr, o.momentum = _opts(), 0.1, 0.9
    muon = lambda: lib.agx_opt_muon(None, m, 1, o, 4096, big)  # noqa: E731
    assert muon() == -1                                             # null arrays
    m[0].w, m[0].g, m[0].m = 4096, 8192, 4096
    assert muon() == -1 and 'different arrays' in err()
    m[0].m = 16384
    o.momentum = 1.0
    assert muon() == -1
    o.momentum, o.lr = 0.9, float('inf')
    assert muon() == -1
    assert lib.agx_opt_muon(None, m, 1, None, 4096, big) == -1


def test_workspace_queries():
    lib = _lib.load()
    small, tall = lib.agx_orth_ws_bytes(_job(), 1, 5), lib.agx_orth_ws_bytes(_job(18161, 256), 1, 5)
    assert 0 < small < tall < 1 << 27
    assert lib.agx_orth_ws_bytes(_job(18161, 256), 1, 3) < tall            # one phase: no intermediate iterate
    assert lib.agx_orth_ws_bytes(_job(), 1, 0) == -1 and lib.agx_orth_ws_bytes(_job(rows=-1), 1, 5) == -1
    assert lib.agx_opt_muon_ws_bytes(None, 1, _lib.MuonOpts()) == -1


def test_oracle_against_singular_values():
    """The iteration maps every singular value by the composed polynomial and keeps the singular vectors."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(9, 5, generator=g, dtype=torch.float64)
    for y in (x, x.t()):
        u, s, v = torch.linalg.svd(y, full_matrices=False)
        s = s / (torch.linalg.vector_norm(y) + 1e-7)
        for _ in range(5):
            s = 3.4445 * s - 4.7750 * s ** 3 + 2.0315 * s ** 5
        assert (N.orthogonalize(y) - u @ torch.diag(s) @ v).abs().max() < 1e-12


def test_matrices_of_a_call_may_not_share_what_is_written():
    """Refused before any launch: two jobs run at once."""
    lib = _lib.load()
    err = lambda: lib.agx_last_error().decode()  # noqa: E731
    big = 1 << 40

    def orth(*ptrs):                                                # (x, out) pairs of 4 x 6 matrices
        j = (_lib.OrthDesc * len(ptrs))()
        for q, (x, out, ld) in zip(j, ptrs):
            q.x, q.out, q.ldx, q.ldo, q.rows, q.cols, q.dtype = x, out, ld, ld, 4, 6, 0
        return lib.agx_orthogonalize(None, j, len(ptrs), _opts(), None, big)
    for bad in ([(4096, 8192, 6), (12288, 8192, 6)], [(4096, 8192, 6), (8192, 12288, 6)], [(4096, 8192, 6), (16384, 8192 + 24 * 3, 6)],
                [(4096, 4096 + 4, 6)], [(4096, 8192, 16), (16384, 8192 + 20, 16)]):
        assert orth(*bad) == -1 and 'overlaps' in err(), bad
    # blocks of columns of one buffer, neighbouring rows of a flat one and one input twice are told apart (workspace missing)
    for good in ([(4096, 4096 + 24, 16)], [(4096, 8192, 6), (4096 + 96, 8192 + 96, 6)], [(4096, 8192, 6), (4096, 12288, 6)]):
        assert orth(*good) == -3, (good, err())

    o = _lib.MuonOpts()
    o.orth, o.lr, o.momentum, o.nesterov = _opts(), 0.1, 0.9, 1

    def muon(*ptrs):
        j = (_lib.MuonDesc * len(ptrs))()
        for q, (w, g, m) in zip(j, ptrs):
            q.w, q.g, q.m, q.ldw, q.ldg, q.ldm, q.rows, q.cols, q.scale = w, g, m, 6, 6, 6, 4, 6, 1.0
        return lib.agx_opt_muon(None, j, len(ptrs), o, None, big)
    for bad in ([(4096, 8192, 12288), (4096, 16384, 20480)], [(4096, 8192, 12288), (20480, 16384, 12288)],
                [(4096, 8192, 12288), (20480, 4096, 24576)], [(4096, 8192, 12288), (20480, 12288, 24576)], [(4096, 4096 + 8, 12288)]):
        assert muon(*bad) == -1 and 'different arrays' in err(), bad
    assert muon((4096, 8192, 12288), (16384, 8192, 20480)) == -3   # one gradient for two kernels is only read


@pytest.mark.parametrize('rows,cols,ld,dtype', [(4, 6, 6, 0), (300, 70, 75, 1)])
def test_workspace_over_a_matrix_is_refused(rows, cols, ld, dtype):
    """Refused before any launch: the call's own workspace over what it reads or writes, from either end."""
    lib = _lib.load()
    mb = 1 << 24
    size = 2 if dtype else 4
    last = ((rows - 1) * ld + cols - 1) * size // 16 * 16
    jobs = lambda cls: (cls * 2)()  # noqa: E731
    j = jobs(_lib.OrthDesc)
    for k, q in enumerate(j):
        q.x, q.out, q.ldx, q.ldo, q.rows, q.cols, q.dtype = (1 + 2 * k) * mb, (2 + 2 * k) * mb, ld, ld, rows, cols, dtype
    n = lib.agx_orth_ws_bytes(j, 2, 5)
    places = [a + d for q in j for a in (q.x, q.out) for d in (0, last, 16 - n)]
    for ws in places:
        assert lib.agx_orthogonalize(None, j, 2, _opts(), ws, n) == -1 and b'workspace overlaps' in lib.agx_last_error(), ws / mb
    o = _lib.MuonOpts()
    o.orth, o.lr, o.momentum, o.nesterov = _opts(), 0.1, 0.9, 1
    m = jobs(_lib.MuonDesc)
    last = ((rows - 1) * ld + cols - 1) * 4 // 16 * 16
    for k, q in enumerate(m):
        q.w, q.g, q.m, q.ldw, q.ldg, q.ldm, q.rows, q.cols, q.scale = *((1 + 3 * k + i) * mb for i in range(3)), ld, ld, ld, rows, cols, 1.0
    n = lib.agx_opt_muon_ws_bytes(m, 2, o)
    for ws in [a + d for q in m for a in (q.w, q.g, q.m) for d in (0, last, 16 - n)]:
        assert lib.agx_opt_muon(None, m, 2, o, ws, n) == -1 and b'workspace overlaps' in lib.agx_last_error(), ws / mb
    if not torch.cuda.is_available():                     # (made-up addresses: what passes would be launched)
        assert lib.agx_orthogonalize(None, j, 2, _opts(), 20 * mb, n) == -2 and lib.agx_opt_muon(None, m, 2, o, 20 * mb, n) == -2
        assert lib.agx_orthogonalize(None, j, 2, _opts(), mb + (last + 256) // 16 * 16, lib.agx_orth_ws_bytes(j, 2, 5)) == -2


@pytest.mark.parametrize('shape,said', [((0, 6), 'no rows'), (((1 << 32) + 4, 2), 'too large'), ((2, (1 << 32) + 4), 'too large'),
                                        ((1 << 31, 1), 'too large')])
def test_refuses_empty_matrices_and_sides_beyond_32_bits(shape, said):
    """Sides go to the library in 32 bits: 2^32 + 4 rows would have been taken for 4."""
    x = torch.empty(*shape, device='meta')
    for call in (lambda: ops.orthogonalize(x), lambda: ops.orthogonalize([torch.zeros(4, 6), x]), lambda: ops.muon(x, x, x, 0.1)):
        with pytest.raises(ValueError, match=said):
            call()


def test_muon_steps_of_any_number_of_kernels_are_checked_at_once():
    """agx_opt_muon_check: the step's own refusals, over more kernels than a call takes, and nothing is launched."""
    lib = _lib.load()
    mb = 1 << 20
    o = _lib.MuonOpts()
    o.orth, o.lr, o.momentum, o.nesterov = _opts(), 0.1, 0.9, 1

    def jobs(n, **kw):                                     # kw: of the last one
        j = (_lib.MuonDesc * n)()
        for k, q in enumerate(j):
            q.w, q.g, q.m, q.ldw, q.ldg, q.ldm, q.rows, q.cols, q.scale = *((3 * k + i) * mb for i in (1, 2, 3)), 6, 6, 6, 4, 6, 1.0
        for k, v in kw.items():
            setattr(j[n - 1], k, v)
        return j
    check = lambda n, o=o, **kw: lib.agx_opt_muon_check(jobs(n, **kw), n, o)  # noqa: E731
    for n in (1, 16, 17, 40):
        assert check(n) == 0 and check(n, g=2 * mb) == 0   # (one gradient for two kernels is only read)
    for kw in (dict(w=mb), dict(w=3 * mb), dict(w=2 * mb), dict(m=mb), dict(m=2 * mb), dict(m=3 * mb + 92), dict(g=mb), dict(g=3 * mb)):
        assert check(18, **kw) == -1 and b'matrices 0 and 17' in lib.agx_last_error(), kw
    for kw in (dict(rows=0), dict(rows=5000, cols=4097), dict(scale=float('inf')), dict(ldm=5), dict(w=None), dict(g=2 * mb + 1),
               dict(ldg=1 << 23)):
        assert check(18, **kw) == -1, kw
    assert check(0) == -1 and lib.agx_opt_muon_check(None, 1, o) == -1 and lib.agx_opt_muon_check(jobs(1), 1, None) == -1
    o.momentum = 1.0
    assert check(18) == -1
    o.momentum, o.orth.steps = 0.9, 0
    assert check(18) == -1


def test_refusals_of_long_lists_name_the_matrix():
    lib = _lib.load()
    o = _lib.MuonOpts()
    o.orth, o.lr, o.momentum = _opts(), 0.1, 0.9
    for n in (1, 16, 17, 33, 40):
        for kw in (dict(rows=0), dict(rows=5000, cols=4097), dict(ldg=1 << 23), dict(scale=float('nan')), dict(w=1)):
            j = (_lib.MuonDesc * n)()
            for k, q in enumerate(j):
                q.w, q.g, q.m, q.ldw, q.ldg, q.ldm, q.rows, q.cols, q.scale = *(((3 * k + i) << 20) for i in (1, 2, 3)), 6, 6, 6, 4, 6, 1.0
            for k, v in kw.items():
                setattr(j[n - 1], k, v)
            assert lib.agx_opt_muon_check(j, n, o) == -1 and ('matrix %d' % (n - 1)) in lib.agx_last_error().decode(), (n, kw)
