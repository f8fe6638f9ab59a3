"""ops.linear_act (vca_matmul_act / vca_linear_act_bwd: a linear layer with bias, activation and residual in the product's
epilogue, forward and gradients) against 64-bit arithmetic, element by element.

Tolerances (u = 2^-24, e = half an ulp of the tensors' type, finfo.eps / 2; |.| of matrices element by element):
  z      the product: q |x| |w|^T for the operands' own rounding (q = 0 for exact fp32 and 16-bit tensors; split into
         16-bit parts of half-ulp h: the dropped lo lo and the rounding of the two lo parts, 3 h^2, single product:
         2 h + h^2) and (K + 8) u (|x| |w|^T + |b|) for fp32 accumulation in any order
  y      |act'| <= 1.13 times that, 8 u (|z| + 1) for the activation's own evaluation, 2 u (|act| + |r|), and e |y|
  dz     |gy| |act''| (dz + k |z|) with |act''| <= 1.13 for the smooth activations and k half an ulp of the type z is
         kept in (half for bf16, fp32 for fp32 and half), 16 u |gy|; where a kinked activation's |z| is within that of
         its kink the slope may be the other one; and e |dz|
  dx     dz's error times |w|, the product's own error as above, and e |dx|; dw likewise with |x|; db = sum |gy| ... of
         dz before its rounding, M u sum |dz|, and e |db|
Half precision adds its smallest subnormal's half, 2^-25, per rounding."""
import ctypes
import math

import pytest
import torch
import torch.nn.functional as F

gpu = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}
ACTS = {None: lambda z: z * 1.0, 'relu': F.relu, 'leaky0.2': lambda z: F.leaky_relu(z, 0.2), 'tanh': torch.tanh,
        'gelu': F.gelu, 'gelu_tanh': lambda z: F.gelu(z, approximate='tanh'), 'silu': F.silu}


@pytest.fixture(autouse=True)
def _reset_precision():
    yield
    from vcagan_amd import ops
    ops.set_precision('fp32')


def _half(mode):
    return 2.0 ** -11 if mode.startswith('fp16') else 2.0 ** -8


def _split_error(mode, dtype, grad):
    """q of the operands' rounding."""
    if dtype != torch.float32 or mode == 'fp32':
        return 0.0
    h = _half(mode)
    single = mode in ('bf16', 'fp16') or (grad and mode in ('mixed', 'fp16-mixed'))
    return 2 * h + h * h if single else 3 * h * h


def _inputs(M, K, N, dtype, seed, bias=True, res=True):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    x, w = r(M, K).to(dtype).cuda(), (r(N, K) / K ** 0.5).to(dtype).cuda()
    return (x, w, (r(N) * 0.5).to(dtype).cuda() if bias else None, r(M, N).to(dtype).cuda() if res else None,
            r(M, N).to(dtype).cuda())


def _mm(a, b):
    return torch.mm(a.contiguous(), b.contiguous())


def _reference(x, w, b, r, gy, act, mode):
    """{name: (value, bound)} of y, dx, dw, db, dr."""
    t = x.dtype
    e = torch.finfo(t).eps / 2 if t != torch.float32 else U
    tiny = 2.0 ** -25 if t == torch.float16 else 0.0
    sub = 2.0 ** -24 if mode.startswith('fp16') and t == torch.float32 else 0.0     # a split part below half's range
    M, K, N = x.shape[0], x.shape[1], w.shape[0]
    X, W, G = x.double(), w.double(), gy.double()
    q = _split_error(mode, t, False)
    P = _mm(X.abs(), W.abs().t())
    z = _mm(X, W.t())
    if b is not None:
        z, P = z + b.double(), P + b.double().abs()
    ez = (q + (K + 8) * U) * P + sub * (X.abs().sum(1, True) + W.abs().sum(1)[None])
    zz = z.clone().requires_grad_(True)
    h = ACTS[act](zz)
    slope, = torch.autograd.grad(h.sum(), zz)
    h = h.detach()
    y = h if r is None else h + r.double()
    out = {'y': (y, 1.13 * ez + 8 * U * (z.abs() + 1) + 2 * U * (h.abs() + y.abs()) + e * y.abs() + tiny)}
    dz = G * slope
    if act is None:
        eu = torch.zeros_like(dz)
    else:
        off = ez + (2.0 ** -11 * z.abs() + 2.0 ** -25 if t == torch.bfloat16 else U * z.abs())
        eu = (G.abs() * torch.where(z.abs() <= off, 1.0, 0.0) if act in ('relu', 'leaky0.2')
              else 1.13 * G.abs() * off) + 16 * U * G.abs()
    ed = eu + (0.0 if act is None else e * (dz.abs() + eu) + tiny)
    q = _split_error(mode, t, True)
    D = dz.abs() + ed
    dx, dw = _mm(dz, W), _mm(dz.t(), X)
    out['dx'] = (dx, _mm(ed, W.abs()) + (q + (N + 8) * U) * _mm(D, W.abs()) + e * dx.abs() + tiny +
                 sub * (D.sum(1, True) + W.abs().sum(0)[None]))
    out['dw'] = (dw, _mm(ed.t(), X.abs()) + (q + (M + 8) * U) * _mm(D.t(), X.abs()) + e * dw.abs() + tiny +
                 sub * (D.sum(0)[:, None] + X.abs().sum(0)[None]))
    db = dz.sum(0)
    out['db'] = (db, eu.sum(0) + (M + 8) * U * D.sum(0) + e * db.abs() + tiny)
    out['dr'] = (G, torch.zeros_like(G))
    return out


def _check(got, want, what):
    val, tol = want
    off = (got.double().reshape(val.shape) - val).abs() - 1.01 * tol - 1e-30
    assert bool((off <= 0).all()), (what, float(off.max()), float(tol.max()))


def _run(M, K, N, dtype, act, seed, mode='fp32', bias=True, res=True):
    from vcagan_amd import ops
    ops.set_precision(mode)
    x, w, b, r, gy = _inputs(M, K, N, dtype, seed, bias, res)
    want = _reference(x, w, b, r, gy, act, mode)
    with torch.no_grad():
        y0 = ops.linear_act(x, w, b, act=act, residual=r)
    leaves = [t for t in (x, w, b, r) if t is not None]
    for t in leaves:
        t.requires_grad_(True)
    y = ops.linear_act(x, w, b, act=act, residual=r)
    assert y.dtype == dtype and y.shape == (M, N) and torch.equal(y.detach(), y0)
    grads = dict(zip([n for n, t in zip('xwbr', (x, w, b, r)) if t is not None], torch.autograd.grad(y, leaves, gy)))
    _check(y.detach(), want['y'], ('y', M, K, N))
    for n, g in grads.items():
        assert g.dtype == dtype
        _check(g, want['d' + n], ('d' + n, M, K, N))


# rows, reduction, columns: single ones, below and just over every tile and chunk, odd and even, few rows with long
# reductions (split over workgroups), the serving kernel's 16-row edge and wide weights beyond it, the 32-row tiles, 64-row
# tiles with four stages, reductions that each tile begins elsewhere
SHAPES = [(1, 1, 1), (1, 8, 16), (2, 3, 5), (1, 512, 512), (7, 129, 33), (15, 1000, 18), (16, 2048, 40), (17, 2048, 40),
          (64, 64, 64), (127, 32, 129), (128, 64, 128), (129, 65, 127), (200, 1111, 77), (333, 96, 513), (40, 5000, 12),
          (600, 256, 1280), (3, 20000, 70), (16, 9001, 33), (24, 4096, 300), (32, 512, 1280), (31, 1000, 70), (20, 8256, 72),
          (17, 40, 2000), (100, 640, 1300), (128, 72, 136), (9, 8192, 8200), (60, 1064, 8200), (33, 128, 8200), (32, 64, 8256),
          (24, 200, 16384)]


@gpu
@pytest.mark.parametrize('dtype', ['fp32', 'bf16', 'fp16'])
@pytest.mark.parametrize('i', range(len(SHAPES)))
def test_forward_and_gradients(i, dtype):
    M, K, N = SHAPES[i]
    _run(M, K, N, TYPES[dtype], list(ACTS)[i % len(ACTS)], 100 + i, bias=i % 5 != 1, res=i % 3 != 1)


@gpu
@pytest.mark.parametrize('dtype', ['bf16', 'fp16'])
@pytest.mark.parametrize('M,K,N', [(4096, 128, 4096), (3500, 136, 4001), (4104, 200, 4000)])
def test_large_tiles(M, K, N, dtype):
    _run(M, K, N, TYPES[dtype], 'gelu', 7)


@gpu
@pytest.mark.parametrize('mode', ['fp32', 'bf16x3', 'fp16x3'])
@pytest.mark.parametrize('M,K,N', [(2400, 2560, 512), (1801, 1112, 680), (700, 4100, 900), (4800, 516, 1280)])
def test_fp32_sizes_between_the_tiles(M, K, N, mode):
    """Tiles that do not divide over the compute units, with and without a split reduction."""
    _run(M, K, N, torch.float32, 'silu', 11, mode=mode)


@gpu
@pytest.mark.parametrize('act', ['relu', 'leaky0.2'])
@pytest.mark.parametrize('M,K,N,dtype,mode', [
    (2400, 2560, 512, 'fp32', 'fp32'), (4800, 512, 1280, 'fp32', 'fp32'), (4800, 1280, 512, 'fp32', 'fp32'),
    (900, 700, 1300, 'fp32', 'fp32'), (2400, 2560, 512, 'fp32', 'bf16x3'), (4800, 512, 1280, 'fp32', 'bf16x3'),
    (4800, 516, 1280, 'fp32', 'fp16x3'), (4800, 512, 1280, 'fp32', 'mixed'), (4096, 128, 4096, 'bf16', 'fp32'),
    (3500, 136, 4001, 'bf16', 'fp32'), (4104, 200, 4000, 'fp16', 'fp32')])
def test_kinked_activations_through_the_tall_and_the_large_tiles(M, K, N, dtype, mode, act):
    _run(M, K, N, TYPES[dtype], act, 13, mode)


@gpu
@pytest.mark.parametrize('dtype', ['fp32', 'bf16', 'fp16'])
@pytest.mark.parametrize('act', list(ACTS))
def test_activations(act, dtype):
    _run(70, 48, 90, TYPES[dtype], act, 5)
    _run(3, 200, 50, TYPES[dtype], act, 6)


@gpu
@pytest.mark.parametrize('mode', ['bf16x3', 'bf16', 'mixed', 'fp16x3', 'fp16', 'fp16-mixed'])
@pytest.mark.parametrize('M,K,N', [(1, 40, 24), (65, 129, 130), (300, 512, 257), (130, 96, 64)])
def test_fp32_tensors_follow_the_precision_mode(M, K, N, mode):
    _run(M, K, N, torch.float32, 'silu', 11, mode)


@gpu
def test_gradient_against_differences():
    from vcagan_amd import ops
    x, w, b, r, gy = _inputs(9, 21, 14, torch.float32, 3)
    for act in (None, 'tanh', 'gelu', 'gelu_tanh', 'silu'):
        ts = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
        f = lambda *a: float((ops.linear_act(*a[:3], act=act, residual=a[3]).double() * gy.double()).sum())
        grads = torch.autograd.grad(ops.linear_act(*ts[:3], act=act, residual=ts[3]), ts, gy)
        h = 2.0 ** -7
        for i, g in enumerate(grads):
            v = torch.randn(ts[i].shape, generator=torch.Generator().manual_seed(i)).cuda()
            with torch.no_grad():
                plus, minus = ([t if j != i else t + s * h * v for j, t in enumerate(ts)] for s in (1, -1))
                diff = (f(*plus) - f(*minus)) / (2 * h)
            # third derivatives are below 2: h^2 / 6 * 2 * sum |gy| |dz|^3, and fp32 noise of the values over h
            step = (v.abs() @ w.abs().t()) if i == 0 else (x.abs() @ v.abs().t()) if i == 1 else v.abs().expand(9, 14)
            tol = float((gy.abs() * (h * h / 3 * step ** 3 + 40 * U * (x.abs() @ w.abs().t() + 4) / h)).sum())
            assert abs(float((g.double() * v.double()).sum()) - diff) <= tol, (act, i)


@gpu
@pytest.mark.parametrize('dtype', ['fp32', 'bf16', 'fp16'])
def test_strides_alignment_and_leading_dimensions(dtype):
    """Rows inside a wider matrix, starts off any vector's alignment, a transposed weight, a broadcast residual, 3-D
    inputs, an expanded incoming gradient: the results are those of dense copies, bit for bit."""
    from vcagan_amd import ops
    t = TYPES[dtype]
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g).to(t).cuda()
    for lead, K, N in (((3, 11), 72, 40), ((2, 2, 5), 33, 19), ((160,), 130, 136)):
        big = r(*lead, K + 9)
        x = big[..., 3:3 + K]
        w = r(K, N).t()
        b = r(2 * N)[1:2 * N:2]
        for res in (r(N).expand(*lead, N), r(*lead, 2 * N)[..., N:], r(*lead[::-1], N).permute(
                *range(len(lead))[::-1], len(lead))):
            dense = [v.detach().clone().contiguous().requires_grad_(True) for v in (x, w, b, res)]
            views = [v.detach().requires_grad_(True) for v in (x, w, b, res)]
            y = ops.linear_act(dense[0], dense[1], dense[2], act='gelu', residual=dense[3])
            v = ops.linear_act(views[0], views[1], views[2], act='gelu', residual=views[3])
            assert y.shape == lead + (N,) and torch.equal(y, v)
            gy = r(N).expand(*lead, N)
            for a, c in zip(torch.autograd.grad(y, dense, gy.contiguous()), torch.autograd.grad(v, views, gy)):
                assert torch.equal(a, c)
    # a residual that broadcasts takes the sum of the rows' gradients
    row = r(N).requires_grad_(True)
    y = ops.linear_act(r(9, K), r(N, K), residual=row.expand(9, N))
    y.sum().backward()
    assert torch.equal(row.grad, torch.full_like(row, 9.0))


@gpu
def test_empty_and_single():
    from vcagan_amd import ops
    x = torch.zeros(0, 12, device='cuda', requires_grad=True)
    w = torch.randn(7, 12).cuda().requires_grad_(True)
    b = torch.randn(7).cuda().requires_grad_(True)
    y = ops.linear_act(x, w, b, act='relu', residual=torch.zeros(0, 7, device='cuda'))
    assert y.shape == (0, 7)
    y.sum().backward()
    assert x.grad.shape == (0, 12) and float(w.grad.abs().max()) == 0.0 and float(b.grad.abs().max()) == 0.0
    assert ops.linear_act(torch.zeros(3, 0, 12, device='cuda'), w).shape == (3, 0, 7)
    v = torch.randn(12).cuda()
    assert torch.equal(ops.linear_act(v, w, b).detach(), ops.linear_act(v[None], w, b)[0].detach())


@gpu
@pytest.mark.parametrize('dtype', ['fp32', 'bf16', 'fp16'])
def test_values_that_are_not_finite_stay_in_their_rows(dtype):
    """A NaN or an infinity in a row of x reaches that row of y and nothing else, whatever its neighbours in the tile."""
    from vcagan_amd import ops
    x, w, b, r, _ = _inputs(150, 72, 130, TYPES[dtype], 2)
    clean = ops.linear_act(x, w, b, act='relu', residual=r)
    x[149, 71], x[3, 0] = math.nan, math.inf
    y = ops.linear_act(x, w, b, act='relu', residual=r)
    keep = torch.ones(150, dtype=torch.bool, device='cuda')
    keep[149] = keep[3] = False
    assert torch.equal(y[keep], clean[keep])
    assert bool(y[149].isnan().all()) and bool((y[3].isinf() | (y[3] == r[3])).all())


# rows through each form of the product: the few-row kernel, the small tiles, split reductions, the tall ones' rows and the
# 256-wide tiles, with columns that end inside a tile
KINKED = [(3, 64, 40), (70, 48, 90), (129, 4100, 67), (1801, 128, 680), (3500, 136, 4001)]


@gpu
@pytest.mark.parametrize('dtype', ['fp32', 'bf16'])
@pytest.mark.parametrize('act', ['relu', 'leaky0.2'])
@pytest.mark.parametrize('M,K,N', KINKED)
def test_kinked_slopes_of_small_values(M, K, N, act, dtype):
    """Pre-activations of either sign around 2^-60, far below half's range but well inside that of fp32 and bf16.  Each row
    of w has one entry, +-1, and each x is a power of two, so z is exact and the slopes are known: dx and db (sums of at
    most M slopes that are multiples of an ulp of 0.2f: M u of them) and dw (powers of two of one sign a column times
    slopes) come out within their summation and one rounding."""
    from vcagan_amd import ops
    t = TYPES[dtype]
    g = torch.Generator().manual_seed(M)
    x = torch.ldexp(torch.ones(M, K), torch.randint(-62, -58, (M, K), generator=g))
    x = (x * torch.where(torch.rand(M, K, generator=g) < 0.5, -1.0, 1.0)).to(t).cuda()
    w = torch.zeros(N, K)
    w[torch.arange(N), torch.randint(0, K, (N,), generator=g)] = torch.where(torch.rand(N, generator=g) < 0.5, -1.0, 1.0)
    w = w.to(t).cuda()
    gy = torch.randint(1, 4, (M, N), generator=g).to(t).cuda()
    leaves = [v.requires_grad_(True) for v in (x, w, torch.zeros(N, dtype=t).cuda())]
    y = ops.linear_act(*leaves, act=act)
    got = torch.autograd.grad(y, leaves, gy)
    X, W, G = x.detach().double(), w.detach().double(), gy.double()
    z = _mm(X, W.t())
    low = 0.0 if act == 'relu' else 0.2
    e = torch.finfo(t).eps / 2
    assert bool((z != 0).all()) and bool(((y.detach().double() - torch.where(z > 0, z, low * z)).abs() <= e * z.abs()).all())
    dz = G * torch.where(z > 0, 1.0, low)
    D = dz * (1 + 2 * e)                                   # the slope 0.2f and dz, each rounded once
    for v, want, size, terms in ((got[0], _mm(dz, W), _mm(D, W.abs()), N), (got[1], _mm(dz.t(), X), _mm(D.t(), X.abs()), M),
                                 (got[2], dz.sum(0), D.sum(0), M)):
        assert bool(((v.double() - want).abs() <= (2 * e + (terms + 8) * U) * size + e * want.abs()).all()), act


@gpu
@pytest.mark.parametrize('act,low', [('relu', 0.0), ('leaky0.2', 0.2)])
def test_slopes_at_every_magnitude(act, low):
    """One power of two a row, of both signs, from the smallest normal bf16 value to past the end of half's range."""
    from vcagan_amd import ops
    for name, bottom in (('bf16', -126), ('fp16', -24), ('fp32', -126)):
        t = TYPES[name]
        mag = 2.0 ** torch.arange(bottom, 16, dtype=torch.float64)
        z = torch.cat([mag, -mag, mag * 0])
        x = z.to(t).cuda()[:, None].requires_grad_(True)
        y = ops.linear_act(x, torch.ones(1, 1, dtype=t).cuda(), act=act)
        gx, = torch.autograd.grad(y, x, torch.ones_like(y))
        assert torch.equal(gx[:, 0].cpu(), torch.where(z > 0, 1.0, low).to(t)), name


@gpu
@pytest.mark.parametrize('dtype', ['fp32', 'bf16', 'fp16'])
def test_slopes_at_a_nan(dtype):
    """torch's: relu hands the incoming gradient on, leaky scales it, the smooth ones' gradients are NaN."""
    from vcagan_amd import ops
    t = TYPES[dtype]
    z = torch.tensor([math.nan, 1.0, -1.0], dtype=t)
    for act, fn in ACTS.items():
        x, ref = (z.clone().cuda()[:, None].requires_grad_(True) for _ in range(2))
        gy = torch.tensor([3.0, 5.0, 7.0], dtype=t).cuda()[:, None]
        got, = torch.autograd.grad(ops.linear_act(x, torch.ones(1, 1, dtype=t).cuda(), act=act), x, gy)
        want, = torch.autograd.grad(fn(ref), ref, gy)
        assert torch.equal(got.isnan(), want.isnan()), act
        if act in (None, 'relu', 'leaky0.2'):
            assert torch.equal(got, want), act


def _act64(act, z):
    """(value, slope) of the smooth activations in 64 bits, from the side that does not cancel; on the CPU."""
    if act == 'gelu':
        phi = 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    c, a = math.sqrt(2.0 / math.pi), 0.044715
    k, dk = (z, torch.ones_like(z)) if act == 'silu' else (2 * c * (z + a * z ** 3), 2 * c * (1 + 3 * a * z * z))
    s = 1.0 / (1.0 + torch.exp(-k))
    return z * s, s + z * dk * s / (1.0 + torch.exp(k))


@gpu
@pytest.mark.parametrize('dtype', ['bf16', 'fp16'])
@pytest.mark.parametrize('act', ['gelu', 'gelu_tanh', 'silu'])
def test_small_values_of_the_activations_keep_their_digits(act, dtype):
    """Far out on the negative side the value is a small product, not a difference: y is off by one rounding to its type (and
    half's subnormals), and by the fp32 evaluation's share: at most 16 u, and 6 u of the exponential's argument k (its terms,
    and the factor log2 e), |k| <= 88."""
    from vcagan_amd import ops
    t = TYPES[dtype]
    z = torch.linspace({'gelu': -13.0, 'gelu_tanh': -9.0, 'silu': -80.0}[act], 9.0, 100001).to(t).unique()
    y = ops.linear_act(z.cuda()[:, None], torch.ones(1, 1, dtype=t).cuda(), act=act).double().cpu()[:, 0]
    want = _act64(act, z.double())[0]
    f = torch.finfo(t)
    tol = want.abs() * (f.eps / 2 + (16 + 6 * 88) * U) + f.smallest_normal * f.eps / 2
    assert bool(((y - want).abs() <= tol).all()), z[(y - want).abs() > tol]


@gpu
@pytest.mark.parametrize('act', ['gelu', 'gelu_tanh', 'silu'])
def test_fp32_activations_are_as_good_as_fp32(act):
    """Value and slope of fp32 tensors against 64 bits, relative to their terms.  The exponential is good to 2 u and its
    argument k to 6 u |k| (silu's and gelu's exactly); the rest: sigmoid 8 u, its slope d = s (1 - s) 14 u; the normal tail
    7 u for its polynomial, 3.1 x 2 u for the reciprocal it is taken at, 2 u for e; 1 - q and the product with z 1 u each."""
    from vcagan_amd import ops
    z = torch.linspace({'gelu': -12.5, 'gelu_tanh': -9.5, 'silu': -85.0}[act], 9.0, 300001).unique()
    x = z.cuda()[:, None].requires_grad_(True)
    y = ops.linear_act(x, torch.ones(1, 1).cuda(), act=act)
    gx, = torch.autograd.grad(y, x, torch.ones_like(y))
    y, gx, z = y.detach()[:, 0].cpu().double(), gx[:, 0].cpu().double(), z.double()
    want, slope = _act64(act, z)
    own = torch.where(slope.abs() < 0.25, 2 * slope.abs(), 1.0)      # the last sum's rounding, of a value at most 1.13
    if act == 'gelu':
        phi = want.abs() / z.abs()
        phi[z == 0] = 0.5
        of_value, of_slope = 20.0, 20 * phi + 10 * (slope - phi).abs() + own
    else:
        k = torch.zeros_like(z) if act == 'silu' else 1.6 * (z + 0.044715 * z ** 3).abs()
        s = want.abs() / z.abs()
        s[z == 0] = 0.5
        of_value, of_slope = 10 + 6 * k, (9 + 6 * k) * s + (20 + 6 * k) * (slope - s).abs() + own
    off, tol = (y - want).abs(), of_value * U * want.abs()
    assert bool((off <= tol).all()), float((off - tol).max())
    off = (gx - slope).abs() - of_slope * U
    assert bool((off <= 0).all()), (z[off > 0], off[off > 0])


@gpu
def test_slopes_far_out():
    """The smooth activations' slopes reach 0 and 1 far from the origin instead of 0 x infinity."""
    from vcagan_amd import ops
    z = torch.tensor([-3e38, -1e20, -200.0, -61.0, 61.0, 200.0, 1e20, 3e38]).cuda()[:, None].requires_grad_(True)
    one = torch.ones(1, 1).cuda()
    for act, low in (('gelu', 0.0), ('gelu_tanh', 0.0), ('silu', 0.0), ('tanh', 0.0)):
        y = ops.linear_act(z, one, act=act)
        gz, = torch.autograd.grad(y.sum(), z)
        hi = 0.0 if act == 'tanh' else 1.0
        assert bool((gz[:4].abs() < 1e-24).all()) and torch.equal(gz[4:], torch.full_like(gz[4:], hi)), (act, gz)
        assert bool(y.isfinite().all())


@gpu
@pytest.mark.parametrize('dtype', ['fp32', 'bf16', 'fp16'])
def test_activations_of_infinity(dtype):
    """+infinity under a smooth activation stays infinity with slope one (tanh: 1 and 0), never infinity x 0."""
    from vcagan_amd import ops
    t = TYPES[dtype]
    x = torch.tensor([[math.inf], [1.0], [math.nan]], dtype=t).cuda().requires_grad_(True)
    one = torch.ones(1, 1, dtype=t).cuda()
    for act in ACTS:
        y = ops.linear_act(x, one, act=act)
        gx, = torch.autograd.grad(y, x, torch.ones_like(y))
        top, slope = (1.0, 0.0) if act == 'tanh' else (math.inf, 1.0)
        y = y.detach()
        assert float(y[0]) == top and float(gx[0]) == slope and bool(y[1].isfinite().all()), (act, y, gx)
        assert bool(y[2].isnan().all()), (act, y)


@gpu
def test_rows_of_the_output_beyond_it_stay():
    """Through the C ABI: C with a row stride wider than its rows, and memory behind the last row, are left alone."""
    from vcagan_amd import _lib
    L = _lib.lib()
    for M, K, N in ((5, 64, 24), (150, 64, 70), (130, 2048, 9)):
        x, w, _, _, _ = _inputs(M, K, N, torch.float32, 4)
        c = torch.full((M + 2, N + 5), 7.5, device='cuda')
        d = _lib.MatmulDesc(M, N, K, 0, 0, 0, 0, 0, 0.0, K, K, N + 5, 0)
        d = ctypes.byref(d)
        n = L.vca_matmul_act_ws_floats(d)
        ws = torch.empty(n + 4, device='cuda')
        ws[n:] = 3.25
        assert L.vca_matmul_act(d, x.data_ptr(), w.data_ptr(), None, None, c.data_ptr(), None, ws.data_ptr(), n,
                                torch.cuda.current_stream().cuda_stream) == 0
        assert bool((c[:, N:] == 7.5).all()) and bool((c[M:] == 7.5).all()) and bool((ws[n:] == 3.25).all())
        want = _mm(x.double(), w.double().t())
        assert bool(((c[:M, :N].double() - want).abs() <= (K + 8) * U * _mm(x.double().abs(), w.double().abs().t())).all())


@gpu
def test_direct_gradients_and_input_grads_only():
    from vcagan_amd import ops
    x, w, b, _, gy = _inputs(90, 64, 48, torch.float32, 8)
    p, q = torch.nn.Parameter(w.clone()), torch.nn.Parameter(b.clone())
    x1 = x.clone().requires_grad_(True)
    gx, gw, gb = torch.autograd.grad(ops.linear_act(x1, p, q, act='silu'), (x1, p, q), gy)
    p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
    with ops.direct_param_grad():
        for _ in range(2):
            ops.linear_act(x1, p, q, act='silu').backward(gy)
    assert torch.equal(x1.grad, gx + gx)
    assert float((p.grad - 1 - 2 * gw).abs().max()) <= 4 * U * float(1 + 2 * gw.abs().max())
    assert float((q.grad - 1 - 2 * gb).abs().max()) <= 4 * U * float(1 + 2 * gb.abs().max())
    x2 = x.clone().requires_grad_(True)
    p.grad = q.grad = None
    with ops.input_grads_only():
        ops.linear_act(x2, p, q, act='silu').backward(gy)
    assert torch.equal(x2.grad, gx) and p.grad is None and q.grad is None


@gpu
@pytest.mark.parametrize('dtype', ['fp32', 'bf16', 'fp16'])
@pytest.mark.parametrize('M,K,N', [(60, 64, 48), (600, 600, 600), (300, 1111, 77), (100, 1000, 4000), (1024, 1024, 1024)])
def test_each_gradient_is_the_same_whichever_are_wanted(M, K, N, dtype):
    """dx and dw by one launch or by their own, and with an operand that starts off the other's alignment."""
    from vcagan_amd import ops
    x, w, b, _, gy = _inputs(M, K, N, TYPES[dtype], 12)
    want = _reference(x, w, b, None, gy, 'silu', 'fp32')
    shifted = torch.empty(M * K + 1, dtype=x.dtype, device='cuda')[1:].view(M, K).copy_(x)
    for x1 in (x, shifted):
        x1 = x1.detach().requires_grad_(True)
        w1, b1 = w.detach().requires_grad_(True), b.detach().requires_grad_(True)
        grads = lambda *leaves: torch.autograd.grad(ops.linear_act(x1, w1, b1, act='silu'), leaves, gy)
        gx, gw, gb = grads(x1, w1, b1)
        for g, n in ((gx, 'dx'), (gw, 'dw'), (gb, 'db')):
            _check(g, want[n], (n, M, K, N))
        assert torch.equal(grads(x1)[0], gx) and torch.equal(grads(w1)[0], gw) and torch.equal(grads(b1)[0], gb)
        x2 = x1.detach()
        gw2, gb2 = torch.autograd.grad(ops.linear_act(x2, w1, b1, act='silu'), (w1, b1), gy)
        assert torch.equal(gw2, gw) and torch.equal(gb2, gb)


@gpu
def test_forward_mode_is_refused_and_traces_keep_the_call():
    """A tangent is never dropped without a word, whichever input carries it and with or without gradients enabled, and
    a trace replays the operator on new inputs instead of the traced call's result."""
    from torch.autograd import forward_ad
    from vcagan_amd import ops
    args = _inputs(4, 8, 5, torch.float32, 1)[:4]
    for i in range(4):
        for grad in (True, False):
            with forward_ad.dual_level(), torch.set_grad_enabled(grad):
                dual = [forward_ad.make_dual(t, torch.ones_like(t)) if i == j else t for j, t in enumerate(args)]
                with pytest.raises(NotImplementedError):
                    ops.linear_act(*dual[:3], act='silu', residual=dual[3])
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda x: ops.linear_act(x, args[1]), (args[0],), (args[0],))
    f = torch.jit.trace(lambda x: ops.linear_act(x, *args[1:3], act='silu'), args[0], check_trace=False)
    for s in (2, 3):
        x = _inputs(4, 8, 5, torch.float32, s)[0]
        assert torch.equal(f(x), ops.linear_act(x, *args[1:3], act='silu'))


@gpu
def test_ragged_batches_keep_a_bounded_number_of_sizes(monkeypatch):
    """A row count of its own in every call: what is remembered of them stays bounded, and forgetting changes nothing."""
    from vcagan_amd import ops
    monkeypatch.setattr(ops, '_act_ws', {})
    x, w, b, _, _ = _inputs(300, 1200, 70, torch.float32, 3)
    x.requires_grad_(True)

    def one(m):
        y = ops.linear_act(x[:m], w, b, act='silu')
        return y.detach(), torch.autograd.grad(y, x, torch.ones_like(y))[0]
    want = [one(m) for m in range(1, 300, 7)]
    assert len(ops._act_ws) == 2 * len(want)
    monkeypatch.setattr(ops, '_act_ws', {})
    monkeypatch.setattr(ops, '_ACT_WS_KEPT', 16)
    for m, (y, gx) in zip(range(1, 300, 7), want):
        got = one(m)
        assert torch.equal(got[0], y) and torch.equal(got[1], gx) and len(ops._act_ws) <= 16


@gpu
def test_streams_and_graph_replay():
    """Forward and backward captured together and replayed on new inputs beside eager work of the same shapes."""
    from vcagan_amd import ops
    x, w, b, r, gy = _inputs(40, 1500, 70, torch.bfloat16, 9)
    ts = [t.clone().requires_grad_(True) for t in (x, w, b, r)]

    def one():
        y = ops.linear_act(ts[0], ts[1], ts[2], act='gelu', residual=ts[3])
        return [y.detach()] + list(torch.autograd.grad(y, ts, gy))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = one()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(eager, one()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = one()
    for rep in range(4):
        with torch.no_grad():
            for i, t in enumerate(ts + [gy]):
                t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(9 * rep + i)))
        want = one()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, want)), rep


@gpu
def test_elements_beyond_32_bits():
    """2.2e9 elements of x, y and dz: the last rows come out as the same rows alone do."""
    from vcagan_amd import ops
    M, K, N = 2_800_000, 768, 776
    x = torch.zeros(M, K, device='cuda', dtype=torch.bfloat16)
    g = torch.Generator().manual_seed(1)
    tail = torch.randn(300, K, generator=g).to(torch.bfloat16).cuda()
    x[-300:] = tail
    w = (torch.randn(N, K, generator=g) / 28).to(torch.bfloat16).cuda().requires_grad_(True)
    small = ops.linear_act(tail, w, act='silu')
    y = ops.linear_act(x, w, act='silu')
    # (another tile may add up in another order, and a rounding to bf16 then fall the other way: one ulp, 2^-7)
    assert float((y[-300:] - small).detach().abs().max()) <= 2.0 ** -7 * float(small.detach().abs().max())
    assert float(y[:-300].detach().abs().max()) == 0.0
    gw, = torch.autograd.grad(y, w, torch.ones_like(y))
    ws, = torch.autograd.grad(small, w, torch.ones_like(small))
    assert float((gw - ws).abs().max()) <= 2.0 ** -7 * float(ws.abs().max())      # likewise


@gpu
def test_two_streams_at_once():
    """Calls on two streams share no workspace: interleaved, each gives what it gives alone."""
    from vcagan_amd import ops
    a, b = _inputs(60, 4000, 50, torch.float32, 1), _inputs(60, 4000, 50, torch.float32, 2)
    want = [ops.linear_act(v[0], v[1], v[2], act='gelu', residual=v[3]) for v in (a, b)]
    norms = [ops.grad_norm([v[0], v[1]]) for v in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for i, (s, v) in enumerate(zip(streams, (a, b))):
            with torch.cuda.stream(s):
                got[i].append((ops.linear_act(v[0], v[1], v[2], act='gelu', residual=v[3]), ops.grad_norm([v[0], v[1]])))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) and torch.equal(n, norms[i]) for y, n in got[i])


@gpu
def test_a_training_step_of_the_operators_together():
    """Two fused layers with a residual, the global norm of their gradients, clipping inside the Adam update: parameters
    after three steps against 64-bit arithmetic.  Tolerance: with exact fp32 products a gradient is off by at most 1e-5
    of its tensor's largest value (reductions of 96 terms: 104 u, twice through the two layers); Adam's update is at
    most 4 lr a step whatever the gradient, and moves by less than lr x 1e-3 where the gradient is over a hundredth of
    the largest one, so the mean deviation is below 1e-3 lr and no element's exceeds 2 lr a step."""
    from vcagan_amd import ops

    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            g = torch.Generator().manual_seed(0)
            self.w1 = torch.nn.Parameter(torch.randn(96, 64, generator=g) / 8)
            self.b1 = torch.nn.Parameter(torch.randn(96, generator=g) / 8)
            self.w2 = torch.nn.Parameter(torch.randn(64, 96, generator=g) / 10)
            self.b2 = torch.nn.Parameter(torch.randn(64, generator=g) / 8)
    net = Net().cuda()
    ref = [p.detach().double() for p in net.parameters()]
    opt = ops.FusedAdam([ops.flatten_module(net)], lr=1e-3)
    flat = [torch.zeros_like(p) for p in ref], [torch.zeros_like(p) for p in ref]
    for t in (1, 2, 3):
        g = torch.Generator().manual_seed(t)
        x, gy = (torch.randn(80, 64, generator=g).cuda() for _ in range(2))
        opt.zero_grad()
        with ops.direct_param_grad():
            y = ops.linear_act(ops.linear_act(x, net.w1, net.b1, act='gelu'), net.w2, net.b2, residual=x)
            y.backward(gy)
        norm = opt.step(max_norm=1.0)
        rp = [p.clone().requires_grad_(True) for p in ref]
        F.linear(F.gelu(F.linear(x.double(), rp[0], rp[1])), rp[2], rp[3]).backward(gy.double())
        total = math.sqrt(sum(float(p.grad.pow(2).sum()) for p in rp))
        assert abs(float(norm) - total) <= 1e-5 * total
        for i, p in enumerate(rp):
            gr = p.grad * min(1.0, 1.0 / (total + 1e-6))
            flat[0][i] = 0.9 * flat[0][i] + 0.1 * gr
            flat[1][i] = 0.999 * flat[1][i] + 0.001 * gr * gr
            ref[i] = ref[i] - 1e-3 / (1 - 0.9 ** t) * flat[0][i] / ((flat[1][i] / (1 - 0.999 ** t)).sqrt() + 1e-8)
    for p, q in zip(net.parameters(), ref):
        off = (p.detach().double() - q).abs()
        assert float(off.mean()) <= 1e-6 and float(off.max()) <= 6e-3


@gpu
def test_each_step_of_the_operators_together():
    """The same network, every step against 64 bits from the parameters and moments the step before it left, so that no
    deviation feeds back.  A gradient is off by at most 4e-5 of its tensor's largest value (three products in a row of at
    most 96 terms, each 104 u of the sum of its terms' magnitudes, itself at most twice the largest), the norm by 4e-5 of
    itself, and the moments and the update follow to first order: with eg the error of c g,
      m  0.1 eg + 3 u (|0.9 m| + |0.1 c g|)        v  0.002 |c g| eg + 0.001 eg^2 + 4 u v
      p  lr' (em / den + |m| ev / (2 sqrt(v) root) / den^2) x 1.5 + 6 u |update| + 2 u |p|
    where v is at least four times its error; that has to be nearly everywhere."""
    from vcagan_amd import ops

    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            g = torch.Generator().manual_seed(5)
            self.w1 = torch.nn.Parameter(torch.randn(96, 64, generator=g) / 8)
            self.b1 = torch.nn.Parameter(torch.randn(96, generator=g) / 8)
            self.w2 = torch.nn.Parameter(torch.randn(64, 96, generator=g) / 10)
            self.b2 = torch.nn.Parameter(torch.randn(64, generator=g) / 8)
    net = Net().cuda()
    (flat, grad), = groups = [ops.flatten_module(net)]
    opt = ops.FusedAdam(groups, lr=1e-3)
    near = 0
    for t in (1, 2, 3):
        g = torch.Generator().manual_seed(10 + t)
        x, gy = (torch.randn(80, 64, generator=g).cuda() for _ in range(2))
        p, m, v = (a.double().clone() for a in (flat, opt.state[0]['m'], opt.state[0]['v']))
        rp = [q.detach().double().requires_grad_(True) for q in net.parameters()]
        F.linear(F.gelu(F.linear(x.double(), rp[0], rp[1])), rp[2], rp[3]).backward(gy.double())
        opt.zero_grad()
        with ops.direct_param_grad():
            ops.linear_act(ops.linear_act(x, net.w1, net.b1, act='gelu'), net.w2, net.b2, residual=x).backward(gy)
        g64, eg = torch.zeros_like(p), torch.zeros_like(p)
        for q, r in zip(net.parameters(), rp):
            at = (q.data_ptr() - flat.data_ptr()) // 4
            g64[at:at + q.numel()] = r.grad.reshape(-1)
            eg[at:at + q.numel()] = 4e-5 * float(r.grad.abs().max())
        assert bool(((grad.double() - g64).abs() <= eg).all())
        total = float(g64.pow(2).sum().sqrt())
        norm = opt.step(max_norm=total * 0.3 * t)              # in force every step, by a factor of its own
        assert abs(float(norm) - total) <= 4e-5 * total
        c = min(1.0, total * 0.3 * t / (total + 1e-6))
        g64, eg = c * g64, c * (eg + 4e-5 * g64.abs())
        em = 0.1 * eg + 3 * U * (0.9 * m.abs() + 0.1 * g64.abs())
        m = 0.9 * m + 0.1 * g64
        v = 0.999 * v + 0.001 * g64 * g64
        ev = 0.002 * g64.abs() * eg + 0.001 * eg * eg + 4 * U * v
        st = opt.state[0]
        assert bool(((st['m'].double() - m).abs() <= em).all()) and bool(((st['v'].double() - v).abs() <= ev).all())
        rate, root = 1e-3 / (1 - 0.9 ** t), math.sqrt(1 - 0.999 ** t)
        den = v.sqrt() / root + 1e-8
        upd = rate * m / den
        tol = (1.5 * rate * (em / den + m.abs() * ev / (2 * v.sqrt() * root).clamp_min(1e-30) / den ** 2) +
               6 * U * upd.abs() + 2 * U * p.abs())
        sure = (4 * ev <= v) | (v == 0)                        # (v == 0: the padding)
        near += int((~sure).sum())
        assert bool(((flat.double() - (p - upd)).abs() <= tol)[sure].all())
    assert near <= 0.01 * flat.numel()


@gpu
def test_refusals_on_device_tensors():
    from vcagan_amd import ops
    x, w, b, r, _ = _inputs(6, 12, 8, torch.float32, 0)
    with pytest.raises(ValueError):
        ops.linear_act(x, w, b, act='swish')
    with pytest.raises(ValueError):
        ops.linear_act(x, w.t())
    with pytest.raises(ValueError):
        ops.linear_act(x, w, b[:7])
    with pytest.raises(ValueError):
        ops.linear_act(x, w, b, residual=r[:1])
    with pytest.raises(ValueError):
        ops.linear_act(x, w.cpu())
    with pytest.raises(ValueError):
        ops.linear_act(torch.zeros(4, 0).cuda(), torch.zeros(3, 0).cuda())
    with pytest.raises(TypeError):
        ops.linear_act(x, w.half())
    with pytest.raises(TypeError):
        ops.linear_act(x.double(), w.double())
    xr = x.requires_grad_(True)
    y = ops.linear_act(xr, w, b, act='tanh')
    g, = torch.autograd.grad(y.sum(), xr, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_packed_structures_are_the_declared_ones():
    from vcagan_amd import _lib
    v = [3, 5, 7, 1, 1, 0, 1, 6, 0.25, 11, 13, 17, 19]
    assert bytes(_lib.MatmulDesc(*v)) == _lib.pack_matmul(*v)
    v = [3, 5, 7, 1, 1, 6, 1, 0, 0.25, 11, 13, 64, 128, 192, 0, 320, 384, 448, 512]
    assert bytes(_lib.LinearBwd(*[None if x == 0 and i > 10 else x for i, x in enumerate(v)])) == _lib.pack_linear_bwd(*v)


def test_remembered_workspace_sizes_are_bounded(monkeypatch):
    from vcagan_amd import ops
    monkeypatch.setattr(ops, '_act_ws', {})
    for m in range(3 * ops._ACT_WS_KEPT):
        assert ops._keep_ws((m, 5), m) == m and ops._act_ws[(m, 5)] == m and len(ops._act_ws) <= ops._ACT_WS_KEPT


def test_refusals_without_a_gpu():
    from vcagan_amd import ops
    with pytest.raises(ValueError):
        ops.linear_act(torch.zeros(2, 4), torch.zeros(3, 4))
    with pytest.raises(TypeError):
        ops.linear_act(torch.zeros(2, 4).double(), torch.zeros(3, 4).double())


def test_entry_points_refuse_before_any_launch():
    from vcagan_amd import _lib
    for elem, own, other in (('bf16', 1, 2), ('fp16', 2, 1)):
        L = _lib.lib(elem)
        ok = dict(M=64, N=64, K=64, type=0, nsplit=0, a_col=0, b_col=0, act=0, slope=0.0, lda=64, ldb=64, ldc=64, ldr=64)
        call = lambda a=64, b=64, c=64, ws=64, n=1 << 30, bias=None, **kw: L.vca_matmul_act(
            ctypes.byref(_lib.MatmulDesc(**dict(ok, **kw))), a, b, bias, None, c, None, ws, n, None)
        for kw in (dict(M=0), dict(N=0), dict(K=0), dict(K=-5), dict(type=3), dict(type=other, nsplit=1),
                   dict(type=own, nsplit=0), dict(type=own, nsplit=3), dict(nsplit=2), dict(act=2), dict(act=8),
                   dict(lda=63), dict(ldb=63), dict(ldc=63), dict(ldr=-1), dict(a_col=1, b_col=0),
                   dict(b_col=1, ldb=63), dict(a_col=1, b_col=1, lda=63), dict(a=None), dict(b=None), dict(c=None),
                   dict(a=66), dict(bias=65)):
            assert call(**kw) == -22, kw
        long = dict(K=1 << 16, lda=1 << 16, ldb=1 << 16)
        n = L.vca_matmul_act_ws_floats(ctypes.byref(_lib.MatmulDesc(**dict(ok, **long))))
        assert n > 0 and n % (64 * 64) == 0
        assert call(ws=None, **long) == -22 and call(n=n - 1, **long) == -22 and call(ws=68, **long) == -22
        bwd = dict(M=64, N=64, K=64, type=0, nsplit=0, act=6, dw_add=0, db_add=0, slope=0.0, ldx=64, ldw=64, gy=64, x=64,
                   w=64, z=64, dz=64, dx=64, dw=64, db=64)
        n = L.vca_linear_act_bwd_ws_floats(ctypes.byref(_lib.LinearBwd(**bwd)))
        assert n > 0
        g = lambda ws=64, n=n, **kw: L.vca_linear_act_bwd(ctypes.byref(_lib.LinearBwd(**dict(bwd, **kw))), ws, n, None)
        for kw in (dict(gy=None), dict(M=0), dict(K=0), dict(act=0), dict(act=2), dict(z=None), dict(dz=None),
                   dict(type=other, nsplit=1), dict(nsplit=2), dict(w=None), dict(x=None), dict(ldx=63), dict(ldw=63),
                   dict(n=n - 1), dict(ws=None), dict(ws=72), dict(N=0), dict(act=9), dict(z=66),
                   dict(type=other, nsplit=1, dx=None, dw=None), dict(act=0, z=None), dict(act=0, dz=None),
                   dict(n=3, dx=None, dw=None), dict(ws=None, n=0, dx=None, dw=None)):
            assert g(**kw) == -22, kw
        assert L.vca_linear_act_bwd_ws_floats(ctypes.byref(_lib.LinearBwd(**dict(bwd, M=0)))) == 0
