"""Global gradient norm, clipping and the clipped Adam update (ops.GradNorm, ops.grad_norm, ops.clip_grad_norm_,
FusedAdam.step(max_norm=), GanStep(max_norm=)) against plain 64-bit arithmetic.

Tolerances.  The kernels hold squares and sums in fp64 and round the norm once: 2^-24 of it, and 2^-30 for the fp64
sums' own order (at most 1e9 terms of 2^-53).  A clipped value is (fp32 factor) x (value): the factor is rounded once
(2^-24), the product once (2^-24) and, in 16-bit types, once more to the type (eps / 2, and half the smallest subnormal
where the result is below the normal range)."""
import ctypes
import math

import numpy as np
import pytest
import torch

gpu = pytest.mark.gpu
F32 = 2.0 ** -24


def _norm64(ts):
    return math.sqrt(sum(float(t.double().pow(2).sum()) for t in ts))


def _list(sizes, dtypes, seed=0, offset=0, scale=1.0):
    """Tensors of the given sizes, dtypes in turn, as views that start `offset` elements behind an aligned address."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for i, n in enumerate(sizes):
        flat = (torch.randn(n + offset + 3, generator=g) * scale).to(dtypes[i % len(dtypes)]).cuda()
        out.append(flat[offset:offset + n])
    return out


def _check_clipped(ts, before, factor):
    for t, b in zip(ts, before):
        want = b.double() * factor
        f = torch.finfo(t.dtype)
        tol = want.abs() * (f.eps / 2 + 2 * F32) + f.smallest_normal * f.eps / 2
        assert bool(((t.double() - want).abs() <= tol).all()), (t.shape, t.dtype)


LISTS = [
    ([1], 0), ([0], 0), ([0, 1, 0, 2, 0], 0), ([7], 1), ([3, 5, 8, 16], 3), ([1023, 1024, 1025], 5),
    ([65536], 0), ([65537, 1], 1), ([4096 * 16 + 3] * 5, 7), ([300000, 17, 1, 999983], 1), ([5] * 161, 2),
    ([513] * 400, 1), ([4000003, 1, 8388608], 3),
]


@gpu
@pytest.mark.parametrize('dtypes', [(torch.float32,), (torch.bfloat16,), (torch.float16,),
                                    (torch.float32, torch.bfloat16, torch.float16)])
@pytest.mark.parametrize('sizes,offset', LISTS)
def test_norm_and_clip(sizes, offset, dtypes):
    from vcagan_amd import ops
    ts = _list(sizes, dtypes, len(sizes), offset)
    guard = [t._base.clone() for t in ts]
    want = _norm64(ts)
    plan = ops.GradNorm(ts)
    got = plan.norm()
    assert got.dtype == torch.float32 and got.shape == ()
    assert abs(float(got) - want) <= want * (F32 + 2.0 ** -30)
    assert float(ops.grad_norm(ts)) == float(got)
    # a bound that is not in force changes nothing; one that is scales every element, and no byte beside the tensors
    for max_norm in (2 * want + 1, math.inf):
        assert float(plan.clip_(max_norm)) == float(got)
        assert all(torch.equal(t._base, b) for t, b in zip(ts, guard))
    max_norm = 0.37 * want
    before = [t.clone() for t in ts]
    assert float(ops.clip_grad_norm_(ts, max_norm)) == float(got)
    _check_clipped(ts, before, min(1.0, max_norm / (want + 1e-6)))
    for t, b in zip(ts, guard):
        n = t.numel()
        assert torch.equal(t._base[:offset], b[:offset]) and torch.equal(t._base[offset + n:], b[offset + n:])
    assert float(plan.clip_(0.0)) >= 0.0
    assert all(float(t.abs().max()) == 0.0 for t in ts if t.numel())


@gpu
@pytest.mark.parametrize('count', [2040, 2048, 2049, 5000])
def test_lists_of_thousands(count):
    """Below, at and above the number of partial sums that a launch of its own adds up, eagerly and replayed on other
    values beside eager calls: the norm has the bits of the norm alone, and every tensor is scaled once."""
    from vcagan_amd import ops
    sizes = [1 + (37 * i) % 900 for i in range(count)]
    ts = _list(sizes, (torch.float32, torch.bfloat16, torch.float16), 8, 1)
    plan = ops.GradNorm(ts)
    plan.norm()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        replayed = plan.clip_(0.5)
    values = torch.randn(sum(sizes), generator=torch.Generator().manual_seed(1)).cuda()
    for rep in range(4):
        for t, v in zip(ts, (values * (rep + 1)).split(sizes)):       # (the types differ: one by one)
            t.copy_(v)
        before = [t.clone() for t in ts]
        want, alone = _norm64(ts), plan.norm()
        if rep == 0:
            norm = float(plan.clip_(0.5))
        else:
            graph.replay()
            torch.cuda.synchronize()
            norm = float(replayed)
        assert norm == float(alone) and abs(norm - want) <= want * (F32 + 2.0 ** -30), rep
        _check_clipped(ts, before, 0.5 / (want + 1e-6))


@gpu
@pytest.mark.parametrize('scale', [1e-30, 1e-22, 1e18, 1e30])
def test_norm_of_values_whose_squares_leave_the_fp32_range(scale):
    from vcagan_amd import ops
    ts = _list([5000, 70000], (torch.float32, torch.bfloat16), 3, 0, scale)
    want = _norm64(ts)
    assert abs(float(ops.grad_norm(ts)) - want) <= want * (F32 + 2.0 ** -30)


@gpu
@pytest.mark.parametrize('n', [100, 200000])
@pytest.mark.parametrize('bad', [math.inf, -math.inf, math.nan])
def test_gradients_that_are_not_finite(n, bad):
    """An infinite norm multiplies by 0 (0 x inf is a NaN), a NaN norm makes everything one: torch's clip."""
    from vcagan_amd import ops
    ts = _list([n, 33], (torch.float32,), 5)
    ts[0][n // 2] = bad
    ref = [t.clone() for t in ts]
    norm = ops.clip_grad_norm_(ts, 1.0)
    if math.isnan(bad):
        assert math.isnan(float(norm)) and all(bool(t.isnan().all()) for t in ts)
    else:
        assert float(norm) == math.inf
        for t, r in zip(ts, ref):
            assert torch.equal(t.isnan(), r.isinf()) and bool((t[~t.isnan()] == 0).all())


@gpu
def test_dense_layouts_and_an_integer_number_of_bits():
    """Permuted-dense gradients are read as the memory they fill; equal inputs give equal bits, also on another stream;
    the version counter sees the in-place change."""
    from vcagan_amd import ops
    g = torch.Generator().manual_seed(9)
    a = torch.randn(7, 5, 64, 33, generator=g).cuda().to(memory_format=torch.channels_last)
    b = torch.randn(129, 65, generator=g).cuda().t()
    want = _norm64([a, b])
    n0 = ops.grad_norm([a, b])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        n1 = ops.grad_norm([a, b])
    torch.cuda.current_stream().wait_stream(side)
    assert float(n0) == float(n1) and abs(float(n0) - want) <= want * (F32 + 2.0 ** -30)
    before, v = [a.clone(), b.clone()], a._version
    ops.clip_grad_norm_([a, b], 0.5)
    _check_clipped([a, b], before, 0.5 / (want + 1e-6))
    assert a._version > v


@gpu
def test_the_memory_of_a_list_stays_when_a_tensor_gets_other_data():
    from vcagan_amd import ops
    t = torch.full((100000,), 2.0, device='cuda')
    n = ops.GradNorm([t])
    t.data = torch.zeros(100000, device='cuda')
    fill = [torch.full((100000,), 9.0, device='cuda') for _ in range(8)]
    assert float(n.norm()) == float(torch.tensor(400000.0).double().sqrt().float())
    n.clip_(1.0)
    assert bool((t == 0).all()) and all(bool((f == 9).all()) for f in fill)


@gpu
def test_shared_memory_is_that_of_the_list_not_of_its_tensors_later():
    from vcagan_amd import ops
    a = torch.randn(1000).cuda()
    n = ops.GradNorm([a, a[100:200]])
    n.tensors[1].data = torch.zeros(100, device='cuda')
    with pytest.raises(ValueError):
        n.clip_(1.0)
    a, b = (torch.randn(1000).cuda() for _ in range(2))
    before = [a.clone(), b.clone()]
    n, old = ops.GradNorm([a, b]), b.detach()
    b.data = a
    n.clip_(1.0)
    _check_clipped([a, old], before, 1.0 / (_norm64(before) + 1e-6))


@gpu
def test_elements_beyond_32_bits():
    from vcagan_amd import ops
    n = 2 ** 31 + 12345
    t = torch.zeros(n + 1, device='cuda', dtype=torch.bfloat16)[1:]
    t[0], t[2 ** 31 + 5], t[-1] = 3.0, 4.0, 12.0
    assert float(ops.clip_grad_norm_([t], 6.5)) == 13.0
    assert [float(t[i]) for i in (0, 2 ** 31 + 5, n - 1)] == [1.5, 2.0, 6.0]
    assert int((t != 0).sum()) == 3


@gpu
def test_scaled_gradients():
    from vcagan_amd import ops
    ts = _list([777, 50001], (torch.float32,), 2)
    sc = ops.LossScaler(ts[0].device, init_scale=1024.0)
    want = _norm64(ts) / 1024.0
    before = [t.clone() for t in ts]
    assert abs(float(ops.grad_norm(ts, sc)) - want) <= want * (F32 + 2.0 ** -30)
    ops.clip_grad_norm_(ts, want / 4, sc)
    _check_clipped(ts, before, want / 4 / (want + 1e-6))


@gpu
def test_graph_replays_on_new_values():
    from vcagan_amd import ops
    ts = _list([300, 123457, 40], (torch.float32, torch.bfloat16), 4)
    plan = ops.GradNorm(ts)
    ts2 = _list([99], (torch.float32,), 6)
    plan2 = ops.GradNorm(ts2)
    plan.norm()
    torch.cuda.synchronize()
    graphs = []
    for p in (plan, plan2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = p.clip_(0.5)
        graphs.append((g, out))
    for rep in range(4):
        for t in ts + ts2:
            t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(rep)).to(t.dtype))
        before = [t.clone() for t in ts]
        before2 = [t.clone() for t in ts2]
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for tt, bb, out in ((ts, before, graphs[0][1]), (ts2, before2, graphs[1][1])):
            want = _norm64(bb)
            assert abs(float(out) - want) <= want * (F32 + 2.0 ** -30), rep
            _check_clipped(tt, bb, 0.5 / (want + 1e-6))


class _Adam64:
    """The update in 64 bits beside a first-order bound of what fp32 rounding (u = 2^-24 an operation) does to it:
      gr = f g + wd p      f, wd and both products rounded, and the sum: dgr <= 4 u (|f g| + |wd p|) + wd dp, however far
                           the two terms cancel
      m  = b1 m + (1-b1) gr      dm <= b1 dm + (1-b1) dgr + 3 u (|b1 m| + |(1-b1) gr|)
      v  = b2 v + (1-b2) gr^2    dv <= b2 dv + (1-b2) 2 |gr| dgr + 4 u v
      s  = lr' m / (sqrt(v) / root + eps)    ds <= lr' (dm + |m| dden / den) / den + 6 u |s|, dden <= dv / (2 sqrt(v) root)
      p  = p - s                 dp <= dp + ds + u |p|
    (the maximum of amsgrad takes the larger of two bounds); checked with a factor of 1.5 for the higher orders."""

    def __init__(self, p, amsgrad):
        self.p = p.double()
        z = torch.zeros_like(self.p)
        self.m, self.v, self.x = z, z, (z if amsgrad else None)
        self.dp = self.dm = self.dv = self.dx = z

    def step(self, g, t, lr, wd, factor, b1=0.9, b2=0.999, eps=1e-8):
        a, b = g.double() * factor, wd * self.p
        gr = a + b
        dgr = 4 * F32 * (a.abs() + b.abs()) + wd * self.dp
        self.dm = b1 * self.dm + (1 - b1) * dgr + 3 * F32 * (b1 * self.m.abs() + (1 - b1) * gr.abs())
        self.m = b1 * self.m + (1 - b1) * gr
        self.v = b2 * self.v + (1 - b2) * gr * gr
        self.dv = b2 * self.dv + (1 - b2) * 2 * gr.abs() * dgr + 4 * F32 * self.v
        q, dq = self.v, self.dv
        if self.x is not None:
            self.x, self.dx = torch.maximum(self.x, self.v), torch.maximum(self.dx, self.dv)
            q, dq = self.x, self.dx
        root = math.sqrt(1 - b2 ** t)
        den = q.sqrt() / root + eps
        s = lr / (1 - b1 ** t) * self.m / den
        ds = lr / (1 - b1 ** t) * (self.dm + self.m.abs() * dq / (2 * q.sqrt().clamp_min(1e-30) * root) / den) / den
        self.p = self.p - s
        self.dp = self.dp + ds + 6 * F32 * s.abs() + F32 * self.p.abs()


def _adam_pair(sizes, amsgrad, seed=0, wd=1e-2):
    from vcagan_amd import ops
    g = torch.Generator().manual_seed(seed)
    groups = [(torch.randn(n, generator=g).cuda(), torch.randn(n, generator=g).cuda()) for n in sizes]
    opt = ops.FusedAdam(groups, lr=1e-3, weight_decay=wd, amsgrad=amsgrad)
    return opt, groups, [_Adam64(f, amsgrad) for f, _ in groups]


def _check_adam(opt, groups, ref):
    for (f, g), st, r in zip(groups, opt.state, ref):
        for got, want, tol in ((st['m'], r.m, r.dm), (st['v'], r.v, r.dv), (f, r.p, r.dp)):
            assert bool(((got.double() - want).abs() <= 1.5 * tol + 1e-30).all())


@gpu
@pytest.mark.parametrize('amsgrad', [False, True])
@pytest.mark.parametrize('sizes', [[4], [100], [4096, 8], [65540, 4, 1000000], [12] * 32, [3000000, 1200004]])
def test_adam_with_clipping(sizes, amsgrad):
    opt, groups, ref = _adam_pair(sizes, amsgrad, len(sizes))
    for t in (1, 2, 3):
        for i, (_, g) in enumerate(groups):
            g.copy_(torch.randn(g.shape, generator=torch.Generator().manual_seed(10 * t + i)))
        want = _norm64([g for _, g in groups])
        max_norm = want * (0.25 if t != 2 else 4.0)
        kept = [g.clone() for _, g in groups]
        norm = opt.step(max_norm=max_norm)
        assert abs(float(norm) - want) <= want * (F32 + 2.0 ** -30)
        assert all(torch.equal(k, g) for k, (_, g) in zip(kept, groups))       # the gradients stay as they are
        fac = min(1.0, max_norm / (want + 1e-6))
        for r, (_, g) in zip(ref, groups):
            r.step(g, t, 1e-3, 1e-2, fac)
        assert int(opt.t_dev) == t == opt.t
        _check_adam(opt, groups, ref)


@gpu
def test_adam_with_clipping_matches_the_unclipped_update_when_the_bound_is_loose():
    from vcagan_amd import ops
    a, ga, _ = _adam_pair([4096, 400], True, 1)
    b, gb, _ = _adam_pair([4096, 400], True, 1)
    assert a.step(max_norm=math.inf) is not None and b.step() is None
    for (f, _), (h, _) in zip(ga, gb):
        assert float((f - h).abs().max()) <= 1e-3 * 4e-5       # 1.f - 0.999f of the plain launch is off by 1.3e-5


@gpu
def test_adam_with_clipping_and_scaler_skips_an_overflow():
    from vcagan_amd import ops
    opt, groups, ref = _adam_pair([4096, 400], False, 1)
    dev = groups[0][0].device
    sc = ops.LossScaler(dev, init_scale=4.0)
    want = _norm64([g for _, g in groups]) / 4.0
    norm = opt.step(sc, 1, max_norm=want / 2)
    assert abs(float(norm) - want) <= want * (F32 + 2.0 ** -30)
    fac = (want / 2) / (want + 1e-6) / 4.0
    for r, (_, g) in zip(ref, groups):
        r.step(g, 1, 1e-3, 1e-2, fac)
    _check_adam(opt, groups, ref)
    kept = [f.clone() for f, _ in groups]
    groups[1][1][399] = math.inf
    assert float(opt.step(sc, 1, max_norm=want)) == math.inf
    assert [int(v) for v in sc.state[1:3]] == [0, 1] and int(opt.t_dev) == 1
    assert all(torch.equal(k, f) for k, (f, _) in zip(kept, groups))
    sc.update()
    assert sc.value == 2.0 and sc.skipped == 1
    groups[1][1][399] = 1.0
    opt.step(sc, 1, max_norm=want)
    assert int(opt.t_dev) == 2 and not any(torch.equal(k, f) for k, (f, _) in zip(kept, groups))


@gpu
@pytest.mark.parametrize('amsgrad', [False, True])
@pytest.mark.parametrize('sizes', [[4096, 400], [3000000, 1200004]])
@pytest.mark.parametrize('bad', [math.inf, math.nan, 'flag'])
def test_adam_with_clipping_and_scaler_skips_in_both_forms(bad, sizes, amsgrad):
    """Few partial sums (every workgroup adds them up) and many (a launch of its own): a gradient that is not finite, in the
    first or the last group, or a flag that is already up beside finite gradients, changes nothing but the flag; the
    other side's flag, the scale and the step count stay, and the step after it counts from there."""
    from vcagan_amd import ops
    opt, groups, ref = _adam_pair(sizes, amsgrad, 4)
    sc = ops.LossScaler(groups[0][0].device, init_scale=8.0)

    def good(t):
        want = _norm64([g for _, g in groups]) / 8.0
        norm = opt.step(sc, 0, max_norm=want / 2)
        assert abs(float(norm) - want) <= want * (F32 + 2.0 ** -30) and int(opt.t_dev) == t
        for r, (_, g) in zip(ref, groups):
            r.step(g, t, 1e-3, 1e-2, (want / 2) / (want + 1e-6) / 8.0)
        _check_adam(opt, groups, ref)
    good(1)
    state = lambda: [f for f, _ in groups] + [st[k] for st in opt.state for k in ('m', 'v', 'vmax') if st[k] is not None]
    kept = [t.clone() for t in state()]
    for k, at in ((0, 0), (1, sizes[1] - 1)):
        was = groups[k][1][at].clone()
        if bad == 'flag':
            sc.state[1] = 1
        else:
            groups[k][1][at] = bad
        norm = float(opt.step(sc, 0, max_norm=1.0))
        assert math.isfinite(norm) if bad == 'flag' else math.isnan(norm) if bad != bad else norm == math.inf
        assert [int(v) for v in sc.state[1:3]] == [1, 0] and int(opt.t_dev) == 1 and sc.value == 8.0
        assert all(torch.equal(a, b) for a, b in zip(kept, state()))
        groups[k][1][at] = was
        sc.state[1] = 0
    good(2)


@gpu
def test_clipped_adam_refuses_groups_that_share_parameters():
    """The groups are updated by one launch: a buffer that is in two of them would be written by both at once."""
    from vcagan_amd import ops
    f, g = torch.ones(64).cuda(), torch.ones(64).cuda()
    for groups in ([(f, g), (f, g)], [(f[:32], g[:32]), (f[16:48], g[16:48])], [(f[32:], g[32:]), (f, g)]):
        opt = ops.FusedAdam(groups)
        with pytest.raises(ValueError):
            opt.step(max_norm=1.0)
        assert int(opt.t_dev) == 0 and opt.t == 0 and bool((f == 1).all())
    opt = ops.FusedAdam([(f[32:], g[32:]), (f[:32], g[:32])])                   # neighbours; gradients may be shared
    assert abs(float(opt.step(max_norm=1.0)) - 8.0) <= 1e-6 and bool((f != 1).all())
    opt = ops.FusedAdam([(f[32:], g[:32]), (f[:32], g[:32])])
    assert abs(float(opt.step(max_norm=1.0)) - 8.0) <= 1e-6


@gpu
def test_adam_with_clipping_under_graph_replay():
    opt, groups, ref = _adam_pair([70000, 400], True, 3)
    opt.step(max_norm=5.0)
    g1 = [g.clone() for _, g in groups]
    fac = lambda gs: 5.0 / (_norm64(gs) + 1e-6)
    for r, g in zip(ref, g1):
        r.step(g, 1, 1e-3, 1e-2, fac(g1))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = opt.step(max_norm=5.0)
    for t in (2, 3, 4):
        for i, (_, g) in enumerate(groups):
            g.copy_(torch.randn(g.shape, generator=torch.Generator().manual_seed(t + 5 * i)))
        opt.param_groups[0]['lr'] = 1e-3 / t
        opt.sync_lr()
        graph.replay()
        torch.cuda.synchronize()
        gs = [g for _, g in groups]
        assert abs(float(norm) - _norm64(gs)) <= _norm64(gs) * (F32 + 2.0 ** -30)
        for r, g in zip(ref, gs):
            r.step(g, t, 1e-3 / t, 1e-2, fac(gs))
        _check_adam(opt, groups, ref)


@gpu
@pytest.mark.parametrize('prec', ['mixed', 'fp16-mixed'])
def test_gan_step_with_clipping(prec):
    """Both sides of a training step clipped: the norms reported are those of the flat gradient buffers the step left
    behind, an eager step and its captured replay report the same, and a bound of zero with no weight decay keeps every
    weight where it was."""
    from oracle import fixtures
    from vcagan_amd import ops, train_step
    ops.set_precision(prec)
    try:
        b = {k: (v.cuda() if k != 'vid_len' else v) for k, v in fixtures.make_batch(2, 20, 112, 5).items()}
        m = fixtures.fill_models(train_step.build_models(), 300)
        for k in m:
            m[k].cuda().train()
        opts = train_step.build_optimizers(m, weight_decay=0.0)
        step = train_step.GanStep(m, opts, 'grid', max_norm=(0.0, 0.0))
        flats = [f.clone() for o in opts for f, _ in o.groups]
        out = step(b['mel'], b['spec'], b['vid'], b['vid_len'], noise=b['noise'])
        assert all(torch.equal(f, g) for f, (g, _) in zip(flats, [x for o in opts for x in o.groups]))
        s = float(step.scaler.scale[1]) if step.scaler is not None else 1.0
        for key, o in (('g_norm', opts[0]), ('d_norm', opts[1])):
            want = _norm64([o.all_grads]) * s
            assert want > 0 and abs(float(out[key]) - want) <= want * (F32 + 2.0 ** -30), key
        gs = train_step.GraphedStep(step, b['mel'], b['spec'], b['vid'], b['vid_len'], b['noise'], warmup=1)
        for _ in range(2):
            r = gs(b['mel'], b['spec'], b['vid'], None, b['noise'])
            for key, o in (('g_norm', opts[0]), ('d_norm', opts[1])):
                want = _norm64([o.all_grads]) * s
                assert abs(float(r[key]) - want) <= want * (F32 + 2.0 ** -30), key
        one = train_step.GanStep(m, opts, 'grid', max_norm=(1.0, None))
        r = one(b['mel'], b['spec'], b['vid'], b['vid_len'], noise=b['noise'])
        assert 'g_norm' in r and 'd_norm' not in r
    finally:
        ops.set_precision('fp32')


@gpu
def test_refusals_on_device_tensors():
    from vcagan_amd import ops
    a = torch.randn(64, 32).cuda()
    with pytest.raises(TypeError):
        ops.grad_norm([torch.nn.Parameter(a)])
    with pytest.raises(TypeError):
        ops.grad_norm([a.double()])
    with pytest.raises(ValueError):
        ops.grad_norm([a[:, :16]])
    with pytest.raises(ValueError):
        ops.grad_norm([a, a.cpu()])
    with pytest.raises(ValueError):
        ops.clip_grad_norm_([a, a], 1.0)
    with pytest.raises(ValueError):
        ops.clip_grad_norm_([a, a.view(-1)[100:200]], 1.0)
    want = _norm64([a, a])
    assert abs(float(ops.grad_norm([a, a])) - want) <= want * (F32 + 2.0 ** -30)      # counted twice, as listed
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError):
            ops.clip_grad_norm_([a], bad)
    opt = ops.FusedAdam([(torch.zeros(4).cuda(), torch.zeros(4).cuda()) for _ in range(33)])
    with pytest.raises(ValueError):
        opt.step(max_norm=1.0)


class _PlainOptimizer:
    """An optimizer with the training step's interface from before there was any clipping."""

    def __init__(self):
        self.all_grads = torch.zeros(8)
        self.flats, self.calls = {}, []

    def step(self, scaler=None, side=0):
        self.calls.append((scaler, side))
        return 'ignored'


def _gan_step(**kw):
    from vcagan_amd import train_step
    g, d = _PlainOptimizer(), _PlainOptimizer()
    return train_step.GanStep({}, (g, d), 'grid', **kw), g, d


def test_gan_step_without_clipping_calls_its_optimizers_as_before():
    step, g, d = _gan_step()
    step._st = dict(g3=torch.zeros(1))
    out = step.finish()
    assert g.calls == [(None, 1)] and set(out) == {'g3'}
    assert step._update(d, 0, step.d_max_norm) is None and d.calls == [(None, 0)]


def test_gan_step_refuses_a_bound_when_it_is_built():
    for bad in (-1.0, math.nan, (1.0, -2.0), [math.nan, None], (1.0,), (1.0, 2.0, 3.0)):
        with pytest.raises(ValueError):
            _gan_step(max_norm=bad)
    step, _, _ = _gan_step(max_norm=(2, None))
    assert (step.g_max_norm, step.d_max_norm) == (2.0, None)
    assert _gan_step(max_norm=0.5)[0].d_max_norm == 0.5


def test_refusals_of_lists():
    from vcagan_amd import ops
    with pytest.raises(ValueError):
        ops.GradNorm([])
    with pytest.raises(ValueError):
        ops.GradNorm([torch.zeros(4)])


def test_entry_points_refuse_before_any_launch():
    from vcagan_amd import _lib
    L = _lib.lib()
    P = lambda *v: (ctypes.c_void_p * len(v))(*v)
    N = lambda *v: (ctypes.c_longlong * len(v))(*v)
    T = lambda *v: (ctypes.c_int * len(v))(*v)
    big = 1 << 20
    bad = [(1, P(None), N(big), T(0)), (1, P(64), N(-1), T(0)), (1, P(64), N(big), T(3)), (1, P(66), N(big), T(0)),
           (1, P(65), N(big), T(1)), (-1, None, None, None), (1, None, N(big), T(0))]
    for n, p, m, t in bad:
        assert L.vca_grad_norm(n, p, m, t, None, 64, 1 << 20, 64, None) == -22
        assert L.vca_grad_clip(n, p, m, t, 1.0, None, 64, 1 << 20, 64, None) == -22
    ok = (1, P(64), N(big), T(0))
    assert L.vca_grad_norm(*ok, None, None, 1 << 20, 64, None) == -22            # no workspace
    assert L.vca_grad_norm(*ok, None, 64, 10, 64, None) == -22                   # a short one
    assert L.vca_grad_norm(*ok, None, 64, 1 << 20, None, None) == -22            # no output
    assert L.vca_grad_clip(*ok, -1.0, None, 64, 1 << 20, 64, None) == -22
    assert L.vca_grad_clip(*ok, math.nan, None, 64, 1 << 20, 64, None) == -22
    g = lambda **kw: (_lib.AdamGroup * 1)(_lib.AdamGroup(**dict(dict(p=64, g=64, m=64, v=64, vmax=None, n=4), **kw)))
    call = lambda tab, n=1, mx=1.0, sc=None, fl=None: L.vca_adam_clip_f32(
        n, tab, mx, .9, .999, 1e-8, 0., 64, 64, sc, fl, 64, 1 << 20, 64, None)
    for kw in (dict(p=None), dict(g=None), dict(m=68), dict(n=5), dict(n=0), dict(vmax=8)):
        assert call(g(**kw)) == -22, kw
    assert call(g(), n=0) == -22 and call(g(), n=33) == -22 and call(g(), mx=-1.0) == -22
    assert call(g(), sc=64) == -22 and call(g(), fl=64) == -22                   # a scale without its flag, and back
    assert L.vca_grad_norm_ws_doubles(10, None, None, None) >= 10
    assert 0 < L.vca_grad_norm_ws_doubles(*ok) < 2050 and L.vca_grad_norm_ws_doubles(1, P(64), N(9), T(0)) == 0
