"""Layer normalisation without a GPU: refusals of the Python entry points and of the C-ABI, struct mirrors, workspace."""
import ctypes

import pytest
import torch

from adversarial_gene_expression_amd import AgxError, _lib, ops


def _x(rows=4, width=8, dtype=torch.float32):
    return torch.zeros(rows, width, dtype=dtype)


def test_struct_mirrors():
    lib = _lib.load()
    for i, m in enumerate([_lib.NormDesc, _lib.OrthDesc, _lib.OrthOpts, _lib.MuonDesc, _lib.MuonOpts]):
        assert lib.agx_op_sizeof(i) == ctypes.sizeof(m), m.__name__
    assert lib.agx_op_sizeof(5) == -1


@pytest.mark.parametrize('x', [torch.zeros(8), torch.zeros(2, 3, 4), torch.zeros(4, 8, dtype=torch.float64),
                               torch.zeros(4, 8, dtype=torch.float16), torch.zeros(4, 0), torch.zeros(8, 4).t(),
                               torch.zeros(4, 1).expand(4, 8), torch.zeros(1, 8).expand(4, 8)])
def test_layer_norm_refuses_operands(x):
    with pytest.raises(ValueError):
        ops.layer_norm(x)


def test_layer_norm_refuses_arguments():
    x = _x()
    for kw in (dict(eps=0.0), dict(eps=float('nan')), dict(act=2), dict(act=1, slope=-0.1), dict(act=1, slope=1.5),
               dict(gamma=torch.ones(7)), dict(gamma=torch.ones(8, dtype=torch.float64)), dict(beta=torch.ones(8, 1)),
               dict(gamma=torch.ones(16)[::2]), dict(out=_x(4, 9)), dict(out=_x(dtype=torch.bfloat16))):
        with pytest.raises(ValueError):
            ops.layer_norm(x, **kw)


def test_backward_refuses_arguments():
    x, v = _x(), torch.zeros(4)
    for args, kw in (((x, x, None, v), {}), ((x, x, v, None), {}), ((x, x, torch.zeros(5), v), {}), ((_x(3), x, v, v), {}),
                     ((_x(dtype=torch.bfloat16), x, v, v), {}), ((x, x, v, v), dict(act=1)),
                     ((x, x, v, v), dict(act=1, y=_x(4, 9))), ((x, x, v, v, torch.ones(3)), {})):
        with pytest.raises(ValueError):
            ops.layer_norm_backward(*args, **kw)
        with pytest.raises(ValueError):
            ops.layer_norm_backward2(x, *args, **kw)
    with pytest.raises(ValueError):
        ops.layer_norm_backward2(_x(5), x, x, v, v)


def test_no_gpu_is_an_error():
    if torch.cuda.is_available():
        pytest.skip('GPU present')
    with pytest.raises(AgxError):
        ops.layer_norm(_x())


def test_abi_refuses_before_any_launch():
    lib = _lib.load()
    d = _lib.NormDesc()
    d.rows, d.width, d.dtype, d.eps = 4, 8, 0, 1e-3
    assert lib.agx_layernorm_fwd(None, None) == -1
    assert lib.agx_layernorm_fwd(None, d) == -1 and b'x missing' in lib.agx_last_error()
    d.x = d.y = 4096
    d.ldx, d.ldy = 7, 8
    assert lib.agx_layernorm_fwd(None, d) == -1
    d.ldx, d.x = 8, 4098                                  # not aligned to its elements
    assert lib.agx_layernorm_fwd(None, d) == -1
    d.x, d.eps = 4096, 0.0
    assert lib.agx_layernorm_fwd(None, d) == -1
    d.eps, d.dtype = 1e-3, 2
    assert lib.agx_layernorm_fwd(None, d) == -1
    d.dtype, d.width = 0, 0
    assert lib.agx_layernorm_fwd(None, d) == -1
    d.width = 8
    assert lib.agx_layernorm_bwd(None, d) == -1           # dy, statistics missing
    d.dy, d.lddy, d.mean, d.rstd, d.dx, d.lddx = 4096, 8, 4096, 4096, 4096, 8
    d.dgamma = 4096
    assert lib.agx_layernorm_bwd(None, d) == -3           # workspace
    d.dgamma, d.dx = None, None
    assert lib.agx_layernorm_bwd(None, d) == -1           # no output
    d.dbeta, d.u, d.ldu = 4096, 4096, 8
    assert lib.agx_layernorm_bwd2(None, d) == -1          # the second order has no term in beta
    d.dbeta, d.rows, d.dx = None, 0, 4096
    assert lib.agx_layernorm_bwd2(None, d) == 0           # no rows: nothing to do
    d.rows = 0
    assert lib.agx_layernorm_fwd(None, d) == 0


def test_workspace_query():
    lib = _lib.load()
    assert lib.agx_layernorm_ws_floats(0, 8, 0) == 0
    for rows, width in ((1, 1), (5, 257), (100000, 256), (3, 40000)):
        for dt in (0, 1):
            n = lib.agx_layernorm_ws_floats(rows, width, dt)
            assert n % (2 * width) == 0 and 2 * width <= n <= 1024 * 2 * width


def test_workspace_of_a_backward_pass():
    """None for few rows, unless dx goes over an input; parameter gradients over an input vector are refused."""
    lib = _lib.load()
    most = lib.agx_layernorm_ws_floats
    for dt in (0, 1):
        assert lib.agx_layernorm_bwd_ws_floats(0, 8, dt) == 0
        for rows, width in ((1, 1), (32, 256), (1536, 256)):
            assert lib.agx_layernorm_bwd_ws_floats(rows, width, dt) == 0
        # (537 vectors of bf16 a row; as float32 1074, which a group of 1024 threads takes, in two launches)
        assert lib.agx_layernorm_bwd_ws_floats(16, 4297, dt) == (0 if dt else most(16, 4297, dt))
        for rows, width in ((1537, 256), (3, 40000), (1500, 4297), (100000, 5)):
            assert lib.agx_layernorm_bwd_ws_floats(rows, width, dt) == most(rows, width, dt) > 0
    d = _lib.NormDesc()
    d.rows, d.width, d.dtype, d.x, d.dy, d.ldx, d.lddy = 2000, 8, 0, 1 << 20, 1 << 21, 8, 8
    d.mean, d.rstd, d.gamma, d.dx, d.lddx, d.dgamma = 4096, 65536, 32768, 1 << 22, 8, 1 << 23
    assert lib.agx_layernorm_bwd(None, d) == -3
    d.rows, d.dx = 32, 1 << 21                            # over dy
    assert lib.agx_layernorm_bwd(None, d) == -3
    d.dx = 1 << 22
    for over in (32768, 32764, 4096, 65536 + 31 * 4):
        d.dgamma = over
        assert lib.agx_layernorm_bwd(None, d) == -1 and b'parameter gradient' in lib.agx_last_error()
        d.dgamma, d.dbeta = None, over
        assert lib.agx_layernorm_bwd(None, d) == -1 and b'parameter gradient' in lib.agx_last_error()
        d.dbeta = None


def test_results_over_vectors_are_refused():
    lib = _lib.load()
    mb = 1 << 20
    d = _lib.NormDesc()
    d.rows, d.width, d.dtype, d.eps = 40, 8, 0, 1e-3
    d.x, d.dy, d.u, d.ldx, d.lddy, d.ldu, d.ldy, d.lddx, d.ldddy = mb, 2 * mb, 3 * mb, 8, 8, 8, 8, 8, 8
    d.gamma, d.beta, d.mean, d.rstd, d.dgamma, d.ws, d.ws_floats = 4 * mb, 5 * mb, 6 * mb, 7 * mb, 8 * mb, 9 * mb, 1 << 15
    for over in (d.gamma, d.beta + 16, d.mean + 39 * 4, d.rstd, d.dgamma, d.ws + 64):
        for entry, name in ((lib.agx_layernorm_fwd, 'y'), (lib.agx_layernorm_bwd, 'dx'), (lib.agx_layernorm_bwd2, 'dx'),
                            (lib.agx_layernorm_bwd2, 'ddy')):
            d.y = d.dx = d.ddy = None
            setattr(d, name, over)
            assert entry(None, d) == -1 and b'an output matrix overlaps' in lib.agx_last_error(), (hex(over), name)


@pytest.mark.parametrize('on,slope', [(0, 0.0), (1, 0.0), (1, 0.2)])
def test_formulas_against_autograd_and_differences(on, slope):
    """The oracle's closed forms of both backward passes against torch's autograd of the definition and against central
    differences, in float64 (differences of step h leave h^2 of the third derivative: 1e-7 at h = 1e-4 here)."""
    from oracle import norm_oracle as N
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    x, dy, u = r(4, 7).requires_grad_(), r(4, 7).requires_grad_(), r(4, 7)
    ga, be = (1 + 0.3 * r(7)).requires_grad_(), (0.3 * r(7)).requires_grad_()
    eps = 1e-3
    y, mean, rstd = N.forward(x, ga, be, eps, slope, on)
    want = torch.autograd.grad(y, (x, ga, be), dy, create_graph=True)
    det = [t.detach() for t in (dy, x, mean, rstd, ga, y)]
    for a, b in zip(N.backward(*det, slope, on), want):
        assert (a - b).abs().max() < 1e-12
    want2 = torch.autograd.grad(want[0], (dy, x, ga), u)
    for a, b in zip(N.backward2(u, *det, slope, on), want2):
        assert (a - b).abs().max() < 1e-12

    def dx_of(xv, dyv, gv):
        _, mm, rr = N.forward(xv, gv, be.detach(), eps, slope, on)
        return (u * N.backward(dyv, xv, mm, rr, gv, det[5], slope, on)[0]).sum()    # (mask held: derivative of a fixed branch)
    h = 1e-4
    for k, (base, grad) in enumerate(zip((dy, x, ga), N.backward2(u, *det, slope, on))):
        base = base.detach()
        for i in range(base.numel()):
            e = torch.zeros_like(base)
            e.view(-1)[i] = h
            args = [[x.detach(), dy.detach(), ga.detach()], [x.detach(), dy.detach(), ga.detach()]]
            at = {0: 1, 1: 0, 2: 2}[k]
            args[0][at], args[1][at] = base + e, base - e
            fd = (dx_of(*args[0]) - dx_of(*args[1])) / (2 * h)
            assert abs(float(fd - grad.reshape(-1)[i])) < 1e-5


def test_outputs_overlap_inputs_only_as_the_same_matrix():
    """Refused before any launch; rows = 4, width = 6."""
    lib = _lib.load()
    err = lambda: lib.agx_last_error().decode()  # noqa: E731

    def desc(**kw):
        d = _lib.NormDesc()
        d.rows, d.width, d.eps, d.act = 4, 6, 1e-3, 0
        d.ldx = d.lddy = d.ldu = d.ldy = d.lddx = d.ldddy = 8
        d.x, d.dy, d.u, d.y, d.mean, d.rstd = 4096, 8192, 12288, 16384, 20480, 24576
        for k, v in kw.items():
            setattr(d, k, v)
        return d
    assert lib.agx_layernorm_fwd(None, desc(y=4096 + 4)) == -1 and 'overlaps' in err()
    assert lib.agx_layernorm_fwd(None, desc(y=4096, ldy=6)) == -1
    for base in (4096, 8192):
        assert lib.agx_layernorm_bwd(None, desc(dx=base + 32)) == -1 and 'overlaps' in err()
    for base in (4096, 8192, 12288):
        assert lib.agx_layernorm_bwd2(None, desc(ddy=base + 8)) == -1 and 'overlaps' in err()
    assert lib.agx_layernorm_bwd2(None, desc(dx=28672, ddy=28672)) == -1 and 'dx and ddy' in err()
    assert lib.agx_layernorm_bwd(None, desc(dx=16384 + 8, act=1)) == -1 and 'overlaps' in err()


@pytest.mark.parametrize('rows,width', [(40, 8), (2000, 300)])
def test_whatever_a_call_writes_is_its_own(rows, width):
    """Refused before any launch: vectors that a pass writes over its matrices, over each other and inside the workspace, and
    the workspace over what is read.  (The sizes take the backward pass in one launch and in two.)"""
    lib = _lib.load()
    mb = 1 << 26

    def desc(**kw):
        d = _lib.NormDesc()
        d.rows, d.width, d.eps, d.act = rows, width, 1e-3, 1
        d.ldx = d.lddy = d.ldu = d.ldy = d.lddx = d.ldddy = width + 3
        d.x, d.dy, d.u, d.y, d.dx, d.ddy, d.gamma, d.beta, d.mean, d.rstd, d.dgamma, d.dbeta, d.ws = (mb * k for k in range(1, 14))
        d.ws_floats = lib.agx_layernorm_ws_floats(rows, width, 0)
        for k, v in kw.items():
            setattr(d, k, v)
        return d
    at = {k: getattr(desc(), k) for k in ('x', 'dy', 'u', 'y', 'dx', 'ddy', 'gamma', 'beta', 'mean', 'rstd', 'dgamma', 'dbeta', 'ws')}
    last = 4 * ((rows - 1) * (width + 3) + width - 1)                  # bytes to a matrix's last element
    fwd, bwd, bwd2 = lib.agx_layernorm_fwd, lib.agx_layernorm_bwd, lib.agx_layernorm_bwd2
    bad = [(fwd, dict(mean=at['x'])), (fwd, dict(rstd=at['x'] + last)), (fwd, dict(mean=at['gamma'])), (fwd, dict(rstd=at['beta'])),
           (fwd, dict(mean=at['rstd'] + 4 * rows - 4)), (fwd, dict(mean=at['y'] + last))]
    for g in ('dgamma', 'dbeta'):
        bad += [(bwd, {g: at[m]}) for m in ('x', 'dy', 'y', 'dx', 'mean', 'rstd', 'gamma', 'ws')]
        bad += [(bwd, {g: at[m] + last}) for m in ('x', 'dy', 'y', 'dx')]
    bad += [(bwd, dict(dbeta=at['dgamma'])), (bwd, dict(dbeta=at['dgamma'] + 4 * width - 4)), (bwd, dict(dgamma=at['ws'] + 8))]
    bad += [(bwd, dict(ws=at[m])) for m in ('x', 'dy', 'y', 'dx', 'gamma', 'mean', 'rstd')]
    bad += [(bwd2, dict(dbeta=None, dgamma=at[m])) for m in ('x', 'dy', 'u', 'y', 'dx', 'ddy', 'mean', 'rstd', 'gamma', 'ws')]
    bad += [(bwd2, dict(dbeta=None, ws=at[m])) for m in ('x', 'dy', 'u', 'y', 'dx', 'ddy', 'mean', 'rstd', 'gamma')]
    for entry, kw in bad:
        assert entry(None, desc(**kw)) == -1 and b' overlaps ' in lib.agx_last_error(), (entry.__name__, kw, lib.agx_last_error())
    if torch.cuda.is_available():
        return                                                         # (made-up addresses: nothing that passes is launched)
    # what is told apart: neighbours, vectors in the padding behind a matrix's columns, a matrix over an input (no device: -2)
    for entry, kw in ((fwd, dict(mean=at['x'] + last + 4)), (fwd, dict(y=at['x'])), (bwd, dict(dbeta=at['dgamma'] + 4 * width)),
                      (bwd, dict(dx=at['dy'])), (bwd, dict(act=0, dgamma=at['y'])), (bwd2, dict(dbeta=None, dx=at['u'], ddy=at['x'])),
                      (bwd, dict(dgamma=None, dbeta=None, ws=at['x']))):
        assert entry(None, desc(**kw)) == -2, (entry.__name__, kw, lib.agx_last_error())


def test_no_rows_ask_for_nothing():
    """An empty matrix has no address: a backward pass without parameter gradients over it is no missing output."""
    lib = _lib.load()
    d = _lib.NormDesc()
    d.rows, d.width, d.eps, d.ldx, d.lddy, d.ldu, d.ldy, d.lddx, d.ldddy = 0, 8, 1e-3, 8, 8, 8, 8, 8, 8
    for entry in (lib.agx_layernorm_fwd, lib.agx_layernorm_bwd, lib.agx_layernorm_bwd2):
        assert entry(None, d) == 0, entry.__name__
    d.dtype = 7                                           # (what is malformed stays refused)
    for entry in (lib.agx_layernorm_fwd, lib.agx_layernorm_bwd, lib.agx_layernorm_bwd2):
        assert entry(None, d) == -1, entry.__name__
