"""Thin op-level wrappers over the C-ABI (one call = one libagx entry point).

Used by the model ``__call__`` path and by the parity tests; the training step
itself is sequenced in C++ (csrc/cgan.hip) to keep Python out of the hot loop.
All arguments and results are device tensors (torch used as allocations only).
"""
import torch

from . import _dev, _lib
from ._dev import ptr


def gemm(A, B, M, N, K, *, ta=0, tb=0, alpha=1.0, bias=None, addrow=None, act=0, slope=0.0, mask=None,
         out=None, accumulate=False, rowscale=None, rowsq=None, force_cfg=-1, force_splitk=0, use_ws=True,
         interp=None, col_scale=None, col_shift=None, sk_flags=None):
    """out[M, N] = epilogue(alpha * op(A) @ op(B)); leading dimensions are the row strides.
    sk_flags: zero-initialised int32 device tensor of agx_gemm_sk_flag_words() words - allows the stream-K form."""
    lib = _lib.load()
    if out is None:
        out = _dev.empty((M, _dev.r4(N)))
    g = _lib.GemmDesc()
    g.A, g.B, g.C = ptr(A), ptr(B), ptr(out)
    g.M, g.N, g.K = M, N, K
    g.lda, g.ldb, g.ldc = A.stride(0), B.stride(0), out.stride(0)
    g.ta, g.tb = ta, tb
    g.alpha = alpha
    g.bias = ptr(bias)
    if addrow is not None:
        g.addrow, g.addmod, g.ldadd = ptr(addrow), addrow.shape[0], addrow.stride(0)
    g.act, g.slope = act, slope
    if mask is not None:
        g.mask, g.ldmask = ptr(mask), mask.stride(0)
    g.accumulate = int(accumulate)
    g.rowscale = ptr(rowscale)
    g.col_scale, g.col_shift = ptr(col_scale), ptr(col_shift)
    if rowsq is not None:
        g.rowsq, g.rowsq_ld = ptr(rowsq), rowsq.stride(0)
    ws = None
    if use_ws:
        wsf = max(int(lib.agx_gemm_ws_floats(M, N, K)), (force_splitk if force_splitk > 0 else 0) * M * N,
                  M * N if interp is not None else 0)
        ws = _dev.empty(max(wsf, 1))
        g.ws, g.ws_floats = ptr(ws), wsf
    g.force_cfg, g.force_splitk = force_cfg, force_splitk
    if sk_flags is not None:
        g.sk_flags, g.sk_flag_words = ptr(sk_flags), sk_flags.numel()
    if interp is not None:   # (rows, alpha): A = [real; fake], out gets the interpolated block too
        g.interp_rows, g.interp_alpha = interp[0], ptr(interp[1])
    _lib.check(lib.agx_gemm_f32(_dev.stream(), g), 'agx_gemm_f32')
    return out


def dense_bn(x, W, b, M, N, K, *, gamma=None, beta=None, eps=1e-3, slope=0.0, act=1, running=None):
    """Dense + batch-norm + (leaky-)ReLU, the optional stage BASELINE.json's north_star names (the reference has
    no batch-norm, tf_utils.py:85-88: nothing on the parity path calls this).
    running=(mean, var): inference form - statistics folded into a per-feature scale / shift applied in the
    GEMM epilogue, ONE launch.  running=None: batch statistics (biased variance over the M rows, as Keras
    BatchNormalization in training mode): GEMM with bias -> column statistics -> folded affine + activation in
    place.  Returns (y, mean, var) with the statistics used."""
    lib = _lib.load()
    scale, shift = _dev.empty(N), _dev.empty(N)
    if running is not None:
        mean, var = running
        _lib.check(lib.agx_bn_fold(_dev.stream(), ptr(mean), ptr(var), 0, ptr(gamma), ptr(beta), eps, ptr(scale),
                                   ptr(shift), N), 'agx_bn_fold')
        return gemm(x, W, M, N, K, bias=b, act=act, slope=slope, col_scale=scale, col_shift=shift), mean, var
    y = gemm(x, W, M, N, K, bias=b)
    mean, std = _dev.empty(N), _dev.empty(N)
    nws = int(lib.agx_colstats_ws_doubles(M, N))
    ws = _dev.empty(nws, dtype=torch.float64)
    _lib.check(lib.agx_colstats(_dev.stream(), ptr(y), y.stride(0), M, N, ptr(mean), ptr(std), ptr(ws), nws), 'agx_colstats')
    _lib.check(lib.agx_bn_fold(_dev.stream(), ptr(mean), ptr(std), 1, ptr(gamma), ptr(beta), eps, ptr(scale), ptr(shift), N),
               'agx_bn_fold')
    _lib.check(lib.agx_affine_act(_dev.stream(), ptr(y), y.stride(0), M, N, ptr(scale), ptr(shift), act, slope),
               'agx_affine_act')
    return y, mean, std * std


_DTYPES = {torch.float32: _lib.AGX_F32, torch.bfloat16: _lib.AGX_BF16}


def _matrix(t, name, like=None):
    """Row stride of a [rows, cols] operand of the normalisation / update operators; raises on what they do not take."""
    if not isinstance(t, torch.Tensor) or t.dim() != 2:
        raise ValueError('%s must be a 2-D tensor' % name)
    dtype, shape = t.dtype, t.shape
    if dtype not in _DTYPES:
        raise ValueError('%s must be float32 or bfloat16, got %s' % (name, dtype))
    rows, cols = shape
    if cols == 0:
        raise ValueError('%s has no columns' % name)
    if like is not None and (shape != like.shape or dtype is not like.dtype or t.get_device() != like.get_device()):
        raise ValueError('%s must match the first operand: got %s %s on %s, expected %s %s on %s'
                         % (name, tuple(shape), dtype, t.device, tuple(like.shape), like.dtype, like.device))
    step, each = t.stride()
    ld = step if rows > 1 else cols
    if (each != 1 and cols > 1) or ld < cols:
        raise ValueError('%s must have contiguous rows that do not overlap (strides %s)' % (name, t.stride()))
    return ld


def _vector(t, name, n, like):
    """A float32 vector of n entries on the operand's device, or None."""
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise ValueError('%s must be a contiguous float32 vector of %d entries' % (name, n))
    if t.get_device() != like.get_device():
        raise ValueError('%s is on %s, the rows on %s' % (name, t.device, like.device))
    return t.data_ptr()


def _on_current(t):
    """The current stream.  Kernels run on the current device: refuse operands that live elsewhere."""
    i = t.get_device()
    if i < 0 or i != torch.cuda.current_device() or not _lib.is_initialised(i):
        if t.device != _dev.device():
            raise ValueError('operands are on %s, the current device is cuda:%d' % (t.device, torch.cuda.current_device()))
    return _dev.stream(i)


def _rows_like(x):
    """Uninitialised [rows, width] result, rows 16-byte aligned as the package lays matrices out, and its row stride."""
    rows, width = x.shape
    q = 3 if x.dtype is torch.float32 else 7
    ld = (width + q) & ~q
    out = x.new_empty((rows, ld))
    return (out if ld == width else out[:, :width]), ld


def _f32(n, x):
    return torch.empty(n, dtype=torch.float32, device=x.device)


def _norm_desc(x, act, slope):
    d = _lib.NormDesc()
    d.ldx = _matrix(x, 'x')
    if act not in (0, 1) or not 0.0 <= slope <= 1.0:
        raise ValueError('act must be 0 or 1 and slope in [0, 1]: got %r, %r' % (act, slope))
    d.x, d.rows, d.width, d.dtype = x.data_ptr(), x.shape[0], x.shape[1], _DTYPES[x.dtype]
    d.act, d.slope = act, slope
    return d


def layer_norm(x, gamma=None, beta=None, *, eps=1e-3, act=0, slope=0.0, out=None):
    """Layer normalisation of every row of x [rows, width] (float32 or bfloat16), with the (leaky-)ReLU of `slope` behind
    it when act=1: y = act(gamma * (x - mean) * rstd + beta), rstd = 1 / sqrt(var + eps), biased variance (Keras
    LayerNormalization).  gamma / beta: float32 vectors or None (1 / 0).  Returns (y, mean, rstd), the statistics in
    float32 for the backward passes, which read x too.  out: where to write y (x itself is allowed where no backward pass
    follows, another overlap with it is not).  The reference has no normalisation layer (tf_utils.py:85-88)."""
    d = _norm_desc(x, act, slope)
    if not eps > 0.0:
        raise ValueError('eps must be positive, got %r' % (eps,))
    d.gamma, d.beta = _vector(gamma, 'gamma', x.shape[1], x), _vector(beta, 'beta', x.shape[1], x)
    if out is not None:
        d.ldy = _matrix(out, 'out', x)
    stream = _on_current(x)
    if out is None:
        out, d.ldy = _rows_like(x)
    mean, rstd = _f32(d.rows, x), _f32(d.rows, x)
    d.y, d.mean, d.rstd, d.eps = out.data_ptr(), mean.data_ptr(), rstd.data_ptr(), eps
    _lib.check(_lib.load().agx_layernorm_fwd(stream, d), 'agx_layernorm_fwd')
    return out, mean, rstd


def _norm_back(d, dy, x, mean, rstd, gamma, y, act):
    if mean is None or rstd is None:
        raise ValueError('mean and rstd of the forward pass are needed')
    d.lddy, d.dy = _matrix(dy, 'dy', x), dy.data_ptr()
    d.mean, d.rstd = _vector(mean, 'mean', x.shape[0], x), _vector(rstd, 'rstd', x.shape[0], x)
    d.gamma = _vector(gamma, 'gamma', x.shape[1], x)
    if act:
        if y is None:
            raise ValueError('act=1 needs y, the forward result: the derivative is taken from its sign')
        d.ldy, d.y = _matrix(y, 'y', x), y.data_ptr()
    return _on_current(x)


def _norm_ws(d, x, floats):
    n = floats(d.rows, d.width, d.dtype)
    if n == 0:
        return None
    ws = _f32(n, x)
    d.ws, d.ws_floats = ws.data_ptr(), n
    return ws


def layer_norm_backward(dy, x, mean, rstd, gamma=None, *, y=None, act=0, slope=0.0, param_grads=True):
    """Backward of layer_norm: (dx, dgamma, dbeta) for the gradient dy of its result, dx in x's type, the parameter
    gradients (sums over all rows in a fixed order) in float32 or None with param_grads=False.  mean / rstd: what the
    forward returned; y: its result, needed with act=1."""
    lib = _lib.load()
    d = _norm_desc(x, act, slope)
    stream = _norm_back(d, dy, x, mean, rstd, gamma, y, act)
    dx, d.lddx = _rows_like(x)
    d.dx = dx.data_ptr()
    ws = dgamma = dbeta = None
    if param_grads:
        ws = _norm_ws(d, x, lib.agx_layernorm_bwd_ws_floats)
        dgamma, dbeta = _f32(d.width, x), _f32(d.width, x)
        d.dgamma, d.dbeta = dgamma.data_ptr(), dbeta.data_ptr()
    _lib.check(lib.agx_layernorm_bwd(stream, d), 'agx_layernorm_bwd')
    return dx, dgamma, dbeta


def layer_norm_backward2(u, dy, x, mean, rstd, gamma=None, *, y=None, act=0, slope=0.0, param_grads=True):
    """Backward of layer_norm_backward's dx with respect to (dy, x, gamma): u is the gradient that arrives at dx, as under
    a gradient penalty (tf_utils.py:154-171).  Returns (ddy, dx, dgamma)."""
    lib = _lib.load()
    d = _norm_desc(x, act, slope)
    d.ldu, d.u = _matrix(u, 'u', x), u.data_ptr()
    stream = _norm_back(d, dy, x, mean, rstd, gamma, y, act)
    (dx, d.lddx), (ddy, d.ldddy) = _rows_like(x), _rows_like(x)
    d.dx, d.ddy = dx.data_ptr(), ddy.data_ptr()
    ws = dgamma = None
    if param_grads:
        ws = _norm_ws(d, x, lib.agx_layernorm_ws_floats)
        dgamma = _f32(d.width, x)
        d.dgamma = dgamma.data_ptr()
    _lib.check(lib.agx_layernorm_bwd2(stream, d), 'agx_layernorm_bwd2')
    return ddy, dx, dgamma


def colsum(A, r0, r1, H, out=None, accumulate=False):
    lib = _lib.load()
    if out is None:
        out = _dev.zeros(H)
    _lib.check(lib.agx_colsum(_dev.stream(), ptr(A), A.stride(0), r0, r1, H, ptr(out), int(accumulate)), 'agx_colsum')
    return out


def rmsprop(w, g, rms, lr, rho=0.9, eps=1e-7, grad_scale=1.0):
    lib = _lib.load()
    _lib.check(lib.agx_opt_rmsprop(_dev.stream(), ptr(w), ptr(g), ptr(rms), w.numel(), lr, rho, eps, grad_scale),
               'agx_opt_rmsprop')


def adam(w, g, m, v, lr_t, b1=0.9, b2=0.999, eps=1e-7, grad_scale=1.0):
    lib = _lib.load()
    _lib.check(lib.agx_opt_adam(_dev.stream(), ptr(w), ptr(g), ptr(m), ptr(v), w.numel(), lr_t, b1, b2, eps,
                                grad_scale), 'agx_opt_adam')


NEWTON_SCHULZ = (3.4445, -4.7750, 2.0315)   # a, b, c that bring singular values from about 0.01 up near 1 in five steps


def _orth_opts(o, steps, coefficients, eps):
    if int(steps) != steps or not 1 <= steps <= _lib.AGX_ORTH_MAX_STEPS:
        raise ValueError('steps must be an integer in 1..%d, got %r' % (_lib.AGX_ORTH_MAX_STEPS, steps))
    c = list(coefficients)
    if len(c) == 3 and not hasattr(c[0], '__len__'):
        c = [c]
    if len(c) not in (1, steps) or any(len(t) != 3 for t in c):
        raise ValueError('coefficients must be one triple (a, b, c) or one per step')
    o.steps, o.n_coef, o.eps = int(steps), len(c), eps
    for k, v in enumerate(v for t in c for v in t):
        o.coef[k] = v
    return o


def _kernel(t, name, like=None):
    """_matrix of an operand that has rows, and sides that the descriptors' 32 bits hold."""
    ld = _matrix(t, name, like)
    if t.shape[0] == 0:
        raise ValueError('%s has no rows' % name)
    if max(t.shape) >= 1 << 31:
        raise ValueError('%s is too large: %s' % (name, tuple(t.shape)))
    return ld


def orthogonalize(x, *, steps=5, coefficients=NEWTON_SCHULZ, eps=1e-7):
    """Newton-Schulz orthogonalisation of a matrix (float32 or bfloat16), or of each of a list of them: X_0 = x / (|x|_F + eps),
    then `steps` times X <- X (a I + b A + c A^2) with A = X^T X (from the left with A = X X^T where rows < cols).  Products of
    operands of 22 bits, summed in float32, one rounding to x's type at the end: errors are those of the float32 iteration
    relative to the matrix's largest entries; an entry below 2^-16 of the largest is held to 2^-38 of that.  Launches are
    shared by up to 16 matrices, whose sums are then split alike: a result's rounding depends on its companions.  The smaller
    side may be at most 4096.  coefficients: (a, b, c), or one such triple per step."""
    one = isinstance(x, torch.Tensor)
    xs = [x] if one else list(x)
    o = _orth_opts(_lib.OrthOpts(), steps, coefficients, eps)
    lds = [_kernel(t, 'x') for t in xs]
    for t in xs:
        _on_current(t)
    lib, outs = _lib.load(), []
    for lo in range(0, len(xs), _lib.AGX_MAX_ORTH):
        part = xs[lo:lo + _lib.AGX_MAX_ORTH]
        jobs = (_lib.OrthDesc * len(part))()
        for j, t, ld in zip(jobs, part, lds[lo:]):
            out, j.ldo = _rows_like(t)
            outs.append(out)
            j.x, j.out, j.ldx = t.data_ptr(), out.data_ptr(), ld
            j.rows, j.cols, j.dtype = t.shape[0], t.shape[1], _DTYPES[t.dtype]
        n = int(lib.agx_orth_ws_bytes(jobs, len(part), o.steps))
        _lib.check(0 if n >= 0 else n, 'agx_orth_ws_bytes')
        ws = torch.empty(n, dtype=torch.uint8, device=part[0].device)
        _lib.check(lib.agx_orthogonalize(_dev.stream(), jobs, len(part), o, ws.data_ptr(), n), 'agx_orthogonalize')
    return outs[0] if one else outs


def muon(w, g, m, lr, *, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5, coefficients=NEWTON_SCHULZ, eps=1e-7,
         scale=None):
    """One Muon step in place on float32 kernels w [in, out] (or lists of them) with gradients g and momentum buffers m:
    m <- momentum m + g; u = g + momentum m (nesterov) or m; w <- (1 - lr weight_decay) w - lr scale orthogonalize(u).
    scale: default sqrt(max(1, out / in)) per kernel; a number applies to all.  A refused call changes nothing."""
    ws_, gs, ms = ([t] if isinstance(t, torch.Tensor) else list(t) for t in (w, g, m))
    if not len(ws_) == len(gs) == len(ms):
        raise ValueError('w, g and m must be as many: got %d, %d, %d' % (len(ws_), len(gs), len(ms)))
    o = _lib.MuonOpts()
    _orth_opts(o.orth, steps, coefficients, eps)
    o.lr, o.momentum, o.weight_decay, o.nesterov = lr, momentum, weight_decay, int(bool(nesterov))
    lds = []
    for a, b, c in zip(ws_, gs, ms):
        if not isinstance(a, torch.Tensor) or a.dtype != torch.float32:
            raise ValueError('w must be float32')
        lds.append((_kernel(a, 'w'), _kernel(b, 'g', a), _kernel(c, 'm', a)))
    for a in ws_:
        _on_current(a)
    if not ws_:
        return
    # (all that can be refused or run out of memory before the first launch: a step is taken whole or not at all)
    lib, most = _lib.load(), _lib.AGX_MAX_ORTH
    jobs = (_lib.MuonDesc * len(ws_))()
    for j, a, b, c, ld in zip(jobs, ws_, gs, ms, lds):
        j.w, j.g, j.m = a.data_ptr(), b.data_ptr(), c.data_ptr()
        j.ldw, j.ldg, j.ldm = ld
        j.rows, j.cols = a.shape
        j.scale = max(1.0, a.shape[1] / a.shape[0]) ** 0.5 if scale is None else scale
    if len(ws_) > most:
        _lib.check(lib.agx_opt_muon_check(jobs, len(ws_), o), 'agx_opt_muon_check')
    calls = []
    for lo in range(0, len(ws_), most):
        n = min(most, len(ws_) - lo)
        part = (_lib.MuonDesc * n).from_buffer(jobs, lo * _lib.C.sizeof(_lib.MuonDesc))
        size = int(lib.agx_opt_muon_ws_bytes(part, n, o))
        _lib.check(0 if size >= 0 else size, 'agx_opt_muon_ws_bytes')
        calls.append((part, n, size))
    ws = torch.empty(max(size for _, _, size in calls), dtype=torch.uint8, device=ws_[0].device)
    for part, n, size in calls:
        _lib.check(lib.agx_opt_muon(_dev.stream(), part, n, o, ws.data_ptr(), size), 'agx_opt_muon')


def rng(n, seed, offset=0, normal=True):
    lib = _lib.load()
    out = _dev.empty(n)
    fn = lib.agx_rng_normal if normal else lib.agx_rng_uniform
    _lib.check(fn(_dev.stream(), ptr(out), n, seed, offset), 'agx_rng')
    return out


def synchronize():
    torch.cuda.synchronize()
