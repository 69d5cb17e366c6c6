"""Layer normalisation kernels against the float64 formulas on the same inputs.

Tolerances: with e = 2^-24 and S the sum of the absolute terms of a result (oracle `*_size`), an element is a tree of at
most 16 serial additions a lane, 6 levels across a wave and 16 wave sums, each adding e of S, plus a few roundings of the
factors and, for dx of the second order, a product of two such sums: 128 e S covers all of them.  Sums over rows run
serially over a workgroup's rows, then over its groups and the workgroups: e per addition, at most rows of them on the
longest path, counted below.  A result stored in bf16 adds half a step, 2^-8 of its value."""
import pytest
import torch

from oracle import norm_oracle as N

pytestmark = pytest.mark.gpu
E = 2.0 ** -24
EPS = 1e-3

# widths around every change of the row's thread group, for both types: part of a wave, a wave, 256 and 1024 threads, the
# form that reads rows again; odd ones; one value; rows: none, one, fewer than a workgroup holds, more than the grid
SHAPES = [(1, 1), (3, 1), (5, 2), (4, 63), (7, 64), (33, 65), (64, 128), (32, 256), (9, 257), (1536, 256), (17, 512), (6, 513),
          (5, 1024), (4, 1025), (3, 1077), (3, 2048), (2, 2050), (5, 4096), (3, 4297), (2, 8192), (2, 8193), (3, 16384),
          (2, 16400), (2, 18154), (40000, 5), (9000, 129)]


def make(rows, width, dtype, seed, ld_extra=0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device='cuda')  # noqa: E731

    def mat(v):
        t = torch.full((rows, width + ld_extra), 7.0, device='cuda', dtype=dtype)[:, :width]
        t.copy_(v)
        return t
    x = mat(r(rows, width) + 0.5 + 0.5 * r(width))
    return x, mat(r(rows, width)), mat(r(rows, width)), 1 + 0.2 * r(width), 0.2 * r(width)


def half_step(dtype):
    return 2.0 ** -8 if dtype == torch.bfloat16 else 0.0


def near(got, want, size, dtype, factor=128):
    got = N.t64(got)
    bad = (got - want).abs() - (factor * E * size + half_step(dtype) * want.abs() + 1e-38)
    assert bool((bad <= 0).all()), (float(bad.max()), int((bad > 0).sum()))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('rows,width', SHAPES)
def test_forward(gpu, rows, width, dtype):
    from adversarial_gene_expression_amd import ops
    x, _, _, ga, be = make(rows, width, dtype, rows * 7 + width, ld_extra=(rows + width) % 3)
    for on, slope in ((0, 0.0), (1, 0.0), (1, 0.2)):
        y, mean, rstd = ops.layer_norm(x, ga, be, eps=EPS, act=on, slope=slope)
        X, G, B = N.t64(x), N.t64(ga), N.t64(be)
        wy, wm, wr = N.forward(X, G, B, EPS, slope, on)
        assert y.dtype == dtype and y.shape == x.shape
        size = N.forward_size(X, G, B, wr)
        near(y, wy, size, dtype)
        near(mean, wm, X.abs().mean(1), torch.float32)
        # rstd: relative error of the variance (its terms' cancelled size over it), halved by the root
        var = 1 / wr ** 2
        near(rstd, wr, wr * (1 + ((X.abs() + wm.abs()[:, None]) ** 2).mean(1) / var), torch.float32)
    y, _, _ = ops.layer_norm(x)                                  # no parameters, default eps, no activation
    near(y, N.forward(X, G * 0 + 1, B * 0, 1e-3)[0], N.forward_size(X, G * 0 + 1, B * 0, wr), dtype)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('rows,width', SHAPES)
def test_backward(gpu, rows, width, dtype):
    from adversarial_gene_expression_amd import ops
    x, dy, u, ga, be = make(rows, width, dtype, rows * 5 + width, ld_extra=(rows + width) % 2)
    deep = 128 + rows
    for on, slope in ((0, 0.0), (1, 0.2)):
        y, mean, rstd = ops.layer_norm(x, ga, be, eps=EPS, act=on, slope=slope)
        args = [N.t64(t) for t in (dy, x, mean, rstd, ga, y)]
        dx, dg, db = ops.layer_norm_backward(dy, x, mean, rstd, ga, y=y, act=on, slope=slope)
        want, size = N.backward(*args, slope, on), N.backward_size(*args, slope, on)
        near(dx, want[0], size[0], dtype)
        near(dg, want[1], size[1], torch.float32, deep)
        near(db, want[2], size[2], torch.float32, deep)
        dx2, none, _ = ops.layer_norm_backward(dy, x, mean, rstd, ga, y=y, act=on, slope=slope, param_grads=False)
        assert none is None and torch.equal(dx2, dx)
        ddy, d2, dg2 = ops.layer_norm_backward2(u, dy, x, mean, rstd, ga, y=y, act=on, slope=slope)
        want, size = N.backward2(N.t64(u), *args, slope, on), N.backward2_size(N.t64(u), *args, slope, on)
        near(ddy, want[0], size[0], dtype)
        near(d2, want[1], size[1], dtype)
        near(dg2, want[2], size[2], torch.float32, deep)


def test_no_rows_and_results_are_reproducible(gpu):
    from adversarial_gene_expression_amd import ops
    x = torch.zeros(0, 24, device='cuda')
    y, mean, rstd = ops.layer_norm(x)
    assert y.shape == (0, 24) and mean.numel() == rstd.numel() == 0
    dx, dg, db = ops.layer_norm_backward(x, x, mean, rstd)
    assert dx.shape == (0, 24) and not dg.any() and not db.any()
    assert not ops.layer_norm_backward2(x, x, x, mean, rstd)[2].any()
    x, dy, u, ga, be = make(5000, 300, torch.float32, 4)
    y, mean, rstd = ops.layer_norm(x, ga, be, act=1)
    a = ops.layer_norm_backward(dy, x, mean, rstd, ga, y=y, act=1)
    b = ops.layer_norm_backward(dy, x, mean, rstd, ga, y=y, act=1)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize('width', [40, 256, 1025, 20000])
def test_rows_do_not_touch_each_other_and_padding_stays(gpu, width):
    """A row of NaN, one of infinities and one constant row leave the others as they are; columns behind the width keep
    their values; the result may be written over the input."""
    from adversarial_gene_expression_amd import ops
    g = torch.Generator(device='cuda').manual_seed(1)
    buf = torch.randn(9, width + 5, generator=g, device='cuda')
    x = buf[:, :width]
    want = ops.layer_norm(x.contiguous(), act=1)[0]
    keep = buf[:, width:].clone()
    bad = buf.clone()
    bad[2, :width] = float('nan')
    bad[4, 3] = float('inf')
    bad[6, :width] = 2.5
    y, mean, rstd = ops.layer_norm(bad[:, :width], out=bad[:, :width], act=1)
    ok = [0, 1, 3, 5, 7, 8]
    assert torch.equal(y[ok], want[ok]) and y.data_ptr() == bad.data_ptr()
    assert torch.isnan(y[2]).all() and torch.isnan(y[4]).all()
    assert not y[6].any() and abs(float(rstd[6]) - 1e-3 ** -0.5) < 1e-5
    assert torch.equal(bad[:, width:], keep)


def test_captured_forward_and_backward_replay(gpu):
    """Forward, backward and second order recorded into one graph: every replay equals the eager calls on its inputs."""
    from adversarial_gene_expression_amd import ops
    x, dy, u, ga, be = make(200, 256, torch.float32, 9)

    def run():
        y, m, r = ops.layer_norm(x, ga, be, act=1, slope=0.2)
        return [y, *ops.layer_norm_backward(dy, x, m, r, ga, y=y, act=1, slope=0.2),
                *ops.layer_norm_backward2(u, dy, x, m, r, ga, y=y, act=1, slope=0.2)]
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for k in range(4):
        x.add_(0.25)
        dy.mul_(-1.5)
        want = [t.clone() for t in run()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k


def test_side_stream(gpu):
    from adversarial_gene_expression_amd import ops
    x, dy, _, ga, be = make(3000, 512, torch.float32, 2)
    y, m, r = ops.layer_norm(x, ga, be)
    want = ops.layer_norm_backward(dy, x, m, r, ga)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        y2, m2, r2 = ops.layer_norm(x, ga, be)
        got = ops.layer_norm_backward(dy, x, m2, r2, ga)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(y, y2) and all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured_without_an_eager_call_before(gpu):
    """Kernels that no eager call has launched yet, straight into a graph; replays against eager calls behind it."""
    from adversarial_gene_expression_amd import ops
    g = torch.Generator().manual_seed(3)
    x, dy, u = (torch.randn(9, 31000, generator=g).to(torch.bfloat16).to(gpu) for _ in range(3))
    gamma, beta = torch.rand(31000, generator=g).to(gpu), torch.rand(31000, generator=g).to(gpu)
    ops.layer_norm(x[:, :8])                             # (the library itself is initialised)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()

    def run():
        y, mean, rstd = ops.layer_norm(x, gamma, beta, act=1, slope=0.2)
        a = ops.layer_norm_backward(dy, x, mean, rstd, gamma, y=y, act=1, slope=0.2)
        return (y,) + a + ops.layer_norm_backward2(u, dy, x, mean, rstd, gamma, y=y, act=1, slope=0.2)
    with torch.cuda.graph(graph):
        kept = run()
    for k in range(3):
        x.mul_(0.5 + k)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(kept, run()):
            assert torch.equal(a, b)


def check_backward(x, dy, ga, be, slope):
    """The backward pass against the formula; returns its operands and results."""
    from adversarial_gene_expression_amd import ops
    y, mean, rstd = ops.layer_norm(x, ga, be, eps=EPS, act=1, slope=slope)
    args = [N.t64(t) for t in (dy, x, mean, rstd, ga, y)]
    got = ops.layer_norm_backward(dy, x, mean, rstd, ga, y=y, act=1, slope=slope)
    want, size = N.backward(*args, slope, 1), N.backward_size(*args, slope, 1)
    near(got[0], want[0], size[0], x.dtype)
    for k in (1, 2):
        near(got[k], want[k], size[k], torch.float32, 128 + x.shape[0])
    return y, mean, rstd, got


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('width', [1, 7, 60, 257, 600, 1077, 2050, 4297])
def test_backward_in_one_launch_and_in_two(gpu, width, dtype):
    """Rows around those that the columns' workgroups take at once, and around the most that one launch takes."""
    for rows in (1, 2, 255, 256, 257, 1023, 1024, 1025, 1535, 1536, 1537, 2100):
        x, dy, _, ga, be = make(rows, width, dtype, rows + width, ld_extra=(rows + width) % 3)
        check_backward(x, dy, ga, be, 0.2)


@pytest.mark.parametrize('rows,width', [(300, 256), (40, 1077), (2000, 600), (300, 14000), (70, 18154), (20, 33001)])
def test_backward_through_the_c_entry(gpu, rows, width):
    """dx over dy and over x, sums on top of what is there, single outputs: the same values as the plain call."""
    from adversarial_gene_expression_amd import _dev, _lib
    lib = _lib.load()
    x, dy, _, ga, be = make(rows, width, torch.float32, rows)
    x, dy = x.contiguous(), dy.contiguous()
    y, mean, rstd, (dx, dg, db) = check_backward(x, dy, ga, be, 0.1)
    ws = torch.empty(lib.agx_layernorm_ws_floats(rows, width, 0), device='cuda')

    def call(x, dy, dx, dgamma, dbeta, add=0):
        d = _lib.NormDesc()
        d.rows, d.width, d.dtype, d.act, d.slope = rows, width, 0, 1, 0.1
        d.x, d.dy, d.y, d.mean, d.rstd, d.gamma = (t.data_ptr() for t in (x, dy, y, mean, rstd, ga))
        d.ldx, d.lddy, d.ldy, d.lddx = x.stride(0), dy.stride(0), y.stride(0), width if dx is None else dx.stride(0)
        d.dx, d.dgamma, d.dbeta = (None if t is None else t.data_ptr() for t in (dx, dgamma, dbeta))
        d.ws, d.ws_floats, d.accumulate_dx, d.accumulate_params = ws.data_ptr(), ws.numel(), add, add
        _lib.check(lib.agx_layernorm_bwd(_dev.stream(), d), 'agx_layernorm_bwd')
    new = lambda t: torch.full_like(t, 5.0)  # noqa: E731
    # (over an input the sums of the parameter gradients run in another order: both are near the formula)
    args = [N.t64(t) for t in (dy, x, mean, rstd, ga, y)]
    want, size = N.backward(*args, 0.1, 1), N.backward_size(*args, 0.1, 1)
    for over in ('x', 'dy'):
        a, b, g, h = x.clone(), dy.clone(), new(dg), new(db)
        o = a if over == 'x' else b
        call(a, b, o, g, h)
        assert torch.equal(o, dx)
        near(g, want[1], size[1], torch.float32, 128 + rows)
        near(h, want[2], size[2], torch.float32, 128 + rows)
    o, g, h = new(dx), new(dg), new(db)
    call(x, dy, o, g, h, add=1)
    for got, plain in ((o, dx), (g, dg), (h, db)):      # (two roundings of the sum, one of the plain value)
        assert bool(((got - 5.0 - plain).abs() <= 4 * E * (5.0 + plain.abs())).all())
    g, h = new(dg), new(db)
    call(x, dy, None, g, h)
    assert torch.equal(g, dg) and torch.equal(h, db)
    g, o = new(dg), new(dx)
    call(x, dy, o, g, None)
    assert torch.equal(g, dg) and torch.equal(o, dx)
    h = new(db)
    call(x, dy, None, None, h)
    assert torch.equal(h, db)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('width', [4100, 8200, 12001, 14000, 16385, 18154, 20481, 24583, 32768, 32775, 33001, 65600])
def test_wide_rows(gpu, width, dtype):
    """Widths around every change of what a thread holds; one row, a few, more than the partial sums have."""
    from adversarial_gene_expression_amd import ops
    for rows in (1, 5, 300):
        x, dy, u, ga, be = make(rows, width, dtype, rows + width, ld_extra=rows % 3)
        y, mean, rstd, _ = check_backward(x, dy, ga, be, 0.2)
        X, G, B = N.t64(x), N.t64(ga), N.t64(be)
        wy, wm, wr = N.forward(X, G, B, EPS, 0.2, 1)
        near(y, wy, N.forward_size(X, G, B, wr), dtype)
        near(mean, wm, X.abs().mean(1), torch.float32)
        args = [N.t64(t) for t in (u, dy, x, mean, rstd, ga, y)]
        got = ops.layer_norm_backward2(u, dy, x, mean, rstd, ga, y=y, act=1, slope=0.2)
        want, size = N.backward2(*args, 0.2, 1), N.backward2_size(*args, 0.2, 1)
        near(got[0], want[0], size[0], dtype)
        near(got[1], want[1], size[1], dtype)
        near(got[2], want[2], size[2], torch.float32, 128 + rows)


@pytest.mark.parametrize('width', [256, 1077, 6000, 18154, 33001])
def test_second_order_over_its_inputs(gpu, width):
    """ddy over dy and dx over x, or over u: the same values as into matrices of their own."""
    from adversarial_gene_expression_amd import _dev, _lib, ops
    lib = _lib.load()
    rows = 37
    x, dy, u, ga, be = (t.contiguous() for t in make(rows, width, torch.float32, width))
    y, mean, rstd = ops.layer_norm(x, ga, be, eps=EPS, act=1, slope=0.2)
    want = ops.layer_norm_backward2(u, dy, x, mean, rstd, ga, y=y, act=1, slope=0.2)
    ws = torch.empty(lib.agx_layernorm_ws_floats(rows, width, 0), device='cuda')
    for dx_over, ddy_over in (('x', 'dy'), ('u', 'x'), ('dy', 'u')):
        m = {'x': x.clone(), 'dy': dy.clone(), 'u': u.clone()}
        dg = torch.full_like(ga, 3.0)
        d = _lib.NormDesc()
        d.rows, d.width, d.dtype, d.act, d.slope = rows, width, 0, 1, 0.2
        d.x, d.dy, d.u, d.y = m['x'].data_ptr(), m['dy'].data_ptr(), m['u'].data_ptr(), y.data_ptr()
        d.ldx, d.lddy, d.ldu, d.ldy, d.lddx, d.ldddy = width, width, width, y.stride(0), width, width
        d.mean, d.rstd, d.gamma, d.dgamma = mean.data_ptr(), rstd.data_ptr(), ga.data_ptr(), dg.data_ptr()
        d.dx, d.ddy, d.ws, d.ws_floats = m[dx_over].data_ptr(), m[ddy_over].data_ptr(), ws.data_ptr(), ws.numel()
        _lib.check(lib.agx_layernorm_bwd2(_dev.stream(), d), 'agx_layernorm_bwd2')
        assert torch.equal(m[ddy_over], want[0]) and torch.equal(m[dx_over], want[1]) and torch.equal(dg, want[2])


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_no_rows_without_parameter_gradients(gpu, dtype):
    from adversarial_gene_expression_amd import ops
    x, v = torch.zeros(0, 24, device='cuda', dtype=dtype), torch.zeros(0, device='cuda')
    dx, dg, db = ops.layer_norm_backward(x, x, v, v, param_grads=False)
    assert dx.shape == (0, 24) and dx.dtype == dtype and dg is None and db is None
    ddy, dx, dg = ops.layer_norm_backward2(x, x, x, v, v, y=x, act=1, param_grads=False)
    assert ddy.shape == dx.shape == (0, 24) and dg is None


def test_rows_of_more_values_than_a_launch_has_threads(gpu):
    """Two rows of 2^27 + 40 bf16 values, odd stride: 32 threads a column of the parameter gradients would be more than 2^32.
    The values are -1, 0 and 1 and mean / rstd 0 / 1: a thread's sums over a row are integers of at most 2^17 + 1, a wave's
    of 2^23 + 64, all exact, and with random signs so are the workgroup's (below 2^20, asserted of the whole).  What is left is
    a rounding each of a mean, its product, two differences and dn q or the sum over the rows, of values up to 3: 8 * 3 e; and
    half a bf16 step."""
    from adversarial_gene_expression_amd import ops
    n = (1 << 27) + 40
    g = torch.Generator(device='cuda').manual_seed(5)
    mk = lambda: torch.randint(-1, 2, (2, n + 1), generator=g, device='cuda', dtype=torch.int8).to(torch.bfloat16)[:, :n]  # noqa: E731
    x, dy, u = mk(), mk(), mk()
    mean, rstd = torch.zeros(2, device='cuda'), torch.ones(2, device='cuda')

    def means(a, r):
        out = float(a[r].double().mean()), float((a[r].double() * x[r].double()).mean())
        assert max(abs(v) * n for v in out) < 2 ** 20
        return out

    def check(got, want):
        assert float(((got.float() - want).abs() - 2.0 ** -8 * want.abs()).max()) <= 24 * E
    dx, dg, db = ops.layer_norm_backward(dy, x, mean, rstd)
    assert torch.equal(dg, (dy.float() * x.float()).sum(0)) and torch.equal(db, dy.float().sum(0))
    for r in range(2):
        mg, mgh = means(dy, r)
        check(dx[r], dy[r].float() - mg - x[r].float() * mgh)
    ddy, dx2, dg2 = ops.layer_norm_backward2(u, dy, x, mean, rstd)
    total = torch.zeros(n, device='cuda')
    for r in range(2):
        mu, muh = means(u, r)
        q = u[r].float() - mu - x[r].float() * muh
        check(ddy[r], q)
        total += dy[r].float() * q
    assert float((dg2 - total).abs().max()) <= 48 * E
    y, m, s = ops.layer_norm(x, eps=1.0)
    for r in range(2):
        mu = float(x[r].double().mean())
        var = float(((x[r].double() - mu) ** 2).mean())
        # (the mean: an exact sum over n as a float - 2^27 + 40 is none, off by 8 of 2^27, a rounding - and the quotient's own;
        #  the variance: 2^17 + 5 additions of a thread's squares, halved by the root)
        assert abs(float(m[r]) - mu) <= 2 * E * abs(mu) and abs(float(s[r]) - (var + 1) ** -0.5) <= 2.0 ** -7
        check(y[r], (x[r].float() - float(m[r])) * float(s[r]))
