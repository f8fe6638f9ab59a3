"""The operators between a training step's forward pass and its parameter update, and the layer in front of them, as
measured work: a linear layer with bias, activation and residual in its epilogue (forward and gradients), the global
norm of many gradient tensors and clipping by it, and the Adam update that takes the clipping factor along.

`run` computes them in plain torch operations where `own` is false and through the framework's entry points where it
is true; `exact` is the definition in 64 bits.
"""
import math

import numpy as np
import torch

own = False

TYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}
ACTS = ('none', 'relu', 'leaky0.2', 'tanh', 'gelu', 'gelu_tanh', 'silu')
BETA1, BETA2, EPS, LR, DECAY, STEPS = 0.9, 0.999, 1e-8, 1e-4, 1e-5, 10
NORM_EPS = 1e-6


# ----------------------------------------------------------------------------------------------------------------
# the cases
# ----------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one time step of a 512-wide layer, the width of the visual features: the smallest call, latency only
        _linear('linear, one row', 1, 512, 512, 'fp32', 'tanh', True, False, False),
        # a few tokens of a wide feed-forward layer when serving: bound by reading the weights once
        _linear('linear, 8 rows wide', 8, 4096, 16384, 'bf16', 'gelu', True, False, False),
        # 32 clips x 75 frames through a 2560 -> 512 projection (the attention's query width), inference
        _linear('linear, 2400 frames', 2400, 2560, 512, 'fp32', 'leaky0.2', True, True, False),
        # the 512 -> 1280 output projection on padded 150-frame clips, trained in exact fp32
        _linear('linear, fp32 training', 4800, 512, 1280, 'fp32', 'relu', True, True, True),
        # every size odd: valid frames of ragged clips gathered into rows, half precision
        _linear('linear, odd sizes', 1801, 1111, 677, 'fp16', 'silu', True, True, True),
        # the largest: a feed-forward layer over 8192 tokens, forward and all gradients
        _linear('linear, bf16 training', 8192, 4096, 4096, 'bf16', 'gelu', True, True, True),
        # gradients of a small head: few values, latency only
        _tensors('norm', 'norm, small head', 6, 5000, 'fp32', False),
        # gradients of a billion parameters in few large 16-bit buckets
        _tensors('norm', 'norm, bf16 buckets', 9, 1000000007, 'bf16', False),
        # the generator side's 246 parameter tensors, 52 M values, each padded to four values in one flat buffer
        _tensors('clip', 'clip, generator side', 246, 51810275, 'fp32', True),
        # odd tensors packed without padding (starts off any vector's alignment), 16- and 32-bit types mixed
        _tensors('clip', 'clip, odd mixed types', 61, 3141593, 'mixed', False),
        # a small network's update: latency only
        _adam('adam, small network', 1, 100000, False),
        # the generator side's update with its three flat buffers
        _adam('adam, generator side', 3, 51810276, True),
    ]


def draw(rng):
    kind = rng.choice(('linear', 'linear', 'linear', 'norm', 'clip', 'adam'))

    def logs(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if kind == 'linear':
        c = _linear('', logs(1, 6000), logs(8, 4096), logs(8, 4096), rng.choice(('fp32', 'bf16', 'fp16')),
                    rng.choice(ACTS), rng.random() < 0.7, rng.random() < 0.5, rng.random() < 0.6)
    elif kind == 'adam':
        c = _adam('', rng.randint(1, 4), logs(4000, 50000000), rng.random() < 0.5)
    else:
        n = logs(1, 240)
        c = _tensors(kind, '', n, logs(max(2 * n, 1000), 200000000), rng.choice(('fp32', 'bf16', 'mixed')),
                     rng.random() < 0.5)
    del c['name']
    return c


def _linear(name, rows, k, n, dtype, act, bias, residual, train):
    return dict(name=name, op='linear', rows=rows, k=k, n=n, dtype=dtype, act=act, bias=bias, residual=residual,
                train=train)


def _tensors(op, name, count, total, dtype, padded):
    return dict(name=name, op=op, count=count, total=total, dtype=dtype, padded=padded)


def _adam(name, buffers, total, amsgrad):
    return dict(name=name, op='adam', buffers=buffers, total=total, amsgrad=amsgrad)


def _sizes(count, total):
    """`count` sizes, at least one each, spread over several orders of magnitude, that add up to `total`."""
    w = np.exp(np.random.RandomState(count).uniform(0.0, 9.0, count))
    ends = np.arange(1, count + 1) + np.floor(np.cumsum(w) / w.sum() * (total - count)).astype(np.int64)
    ends[-1] = total
    return np.diff(ends, prepend=0)


# ----------------------------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)

    def normal(shape, dtype, scale=1.0):
        return torch.randn(shape, generator=g, device='cuda', dtype=dtype).mul_(scale)
    if case['op'] == 'linear':
        t, m, k, n = TYPES[case['dtype']], case['rows'], case['k'], case['n']
        s = dict(case=case, x=normal((m, k), t), w=normal((n, k), t, 1.0 / math.sqrt(k)),
                 b=normal((n,), t, 0.5) if case['bias'] else None,
                 r=normal((m, n), t) if case['residual'] else None,
                 gy=normal((m, n), t) if case['train'] else None)
        if case['train']:
            for name in ('x', 'w', 'b', 'r'):
                if s[name] is not None:
                    s[name].requires_grad_(True)
        return s
    if case['op'] == 'adam':
        sizes = (_sizes(case['buffers'], case['total']) + 3) // 4 * 4
        s = dict(case=case, p=[normal((int(z),), torch.float32, 0.02) for z in sizes],
                 g=[normal((int(z),), torch.float32, 1e-3) for z in sizes],
                 m=[normal((int(z),), torch.float32, 1e-4) for z in sizes],
                 v=[normal((int(z),), torch.float32, 1e-3).square_() for z in sizes], t=STEPS)
        s['vmax'] = [v * 1.25 for v in s['v']] if case['amsgrad'] else None
        s['max_norm'] = 5e-4 * math.sqrt(float(sizes.sum()))     # half the gradients' norm: the bound is in force
        if own:
            from vcagan_amd import ops
            s['opt'] = ops.FusedAdam(list(zip(s['p'], s['g'])), lr=LR, betas=(BETA1, BETA2), eps=EPS,
                                     weight_decay=DECAY, amsgrad=case['amsgrad'])
            for i, st in enumerate(s['opt'].state):
                st['m'], st['v'] = s['m'][i], s['v'][i]
                st['vmax'] = s['vmax'][i] if case['amsgrad'] else None
            s['opt'].t = STEPS
            s['opt'].t_dev.fill_(STEPS)
        return s
    # gradients as views of flat buffers, one buffer per type; padded: starts at multiples of four values
    sizes = _sizes(case['count'], case['total'])
    kinds = np.arange(case['count']) % 3 == 2 if case['dtype'] == 'mixed' else np.full(case['count'],
                                                                                       case['dtype'] == 'bf16')
    flats, grads = [], [None] * case['count']
    for bf16 in (False, True):
        at = np.nonzero(kinds == bf16)[0]
        if len(at):
            room = (sizes[at] + 3) // 4 * 4 if case['padded'] else sizes[at]
            ends = np.cumsum(room)
            flat = torch.zeros(int(ends[-1]), device='cuda', dtype=torch.bfloat16 if bf16 else torch.float32)
            values = normal(flat.shape, flat.dtype, 1e-2)
            for i, e, z in zip(at, ends, room):
                a = int(e - z)
                grads[i] = flat[a:a + int(sizes[i])]
                grads[i].copy_(values[a:a + int(sizes[i])])
            flats.append(flat)
    s = dict(case=case, flats=flats, grads=grads, max_norm=0.5)
    if own:
        from vcagan_amd import ops
        s['plan'] = ops.GradNorm(grads)
    return s


# ----------------------------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------------------------
def run(s):
    case = s['case']
    if case['op'] == 'linear':
        return _own_linear(s, case) if own else _plain_linear(s, case)
    if case['op'] == 'norm':
        return s['plan'].norm() if own else _plain_norm(s['grads'])
    if case['op'] == 'clip':
        # the bound follows the falling gradient norm of a training run, so that it is in force in every pass
        s['max_norm'] *= 0.999
        norm = s['plan'].clip_(s['max_norm']) if own else _plain_clip(s['grads'], s['max_norm'])
        return dict(norm=norm, grads=s['flats'])
    if own:
        norm = s['opt'].step(max_norm=s['max_norm'])
    else:
        norm = _plain_adam(s)
    return dict(norm=norm, p=s['p'], m=s['m'], v=s['v'], vmax=s['vmax'])


def _own_linear(s, case):
    from vcagan_amd import ops
    act = None if case['act'] == 'none' else case['act']
    if not case['train']:
        with torch.no_grad():
            return dict(y=ops.linear_act(s['x'], s['w'], s['b'], act=act, residual=s['r']))
    names = [k for k in ('x', 'w', 'b', 'r') if s[k] is not None]
    y = ops.linear_act(s['x'], s['w'], s['b'], act=act, residual=s['r'])
    grads = torch.autograd.grad(y, [s[k] for k in names], s['gy'])
    return dict(y=y.detach(), **{'d' + k: g for k, g in zip(names, grads)})


@torch.no_grad()
def _plain_linear(s, case):
    t = TYPES[case['dtype']]
    x, w = s['x'].float(), s['w'].float()
    z = x @ w.t()
    if s['b'] is not None:
        z = z + s['b'].float()
    y = _act(z, case['act'])
    if s['r'] is not None:
        y = y + s['r'].float()
    out = dict(y=y.to(t))
    if case['train']:
        dz = s['gy'].float() * _act_slope(z, case['act'])
        out['dx'], out['dw'] = (dz @ w).to(t), (dz.t() @ x).to(t)
        if s['b'] is not None:
            out['db'] = dz.sum(0).to(t)
        if s['r'] is not None:
            out['dr'] = s['gy']
    return out


_GELU_C, _GELU_A = math.sqrt(2.0 / math.pi), 0.044715


def _act(z, act):
    if act == 'relu':
        return torch.where(z > 0, z, 0.0)
    if act == 'leaky0.2':
        return torch.where(z > 0, z, 0.2 * z)
    if act == 'tanh':
        return torch.tanh(z)
    if act == 'gelu':
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == 'gelu_tanh':
        return 0.5 * z * (1.0 + torch.tanh(_GELU_C * (z + _GELU_A * z * z * z)))
    if act == 'silu':
        return z / (1.0 + torch.exp(-z))
    return z


def _act_slope(z, act):
    if act == 'relu':
        return torch.where(z > 0, 1.0, 0.0).to(z.dtype)
    if act == 'leaky0.2':
        return torch.where(z > 0, 1.0, 0.2).to(z.dtype)
    if act == 'tanh':
        h = torch.tanh(z)
        return 1.0 - h * h
    if act == 'gelu':
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if act == 'gelu_tanh':
        h = torch.tanh(_GELU_C * (z + _GELU_A * z * z * z))
        return 0.5 * (1.0 + h) + 0.5 * z * (1.0 - h * h) * _GELU_C * (1.0 + 3.0 * _GELU_A * z * z)
    if act == 'silu':
        e = 1.0 / (1.0 + torch.exp(-z))
        return e * (1.0 + z * (1.0 - e))
    return torch.ones_like(z)


def _plain_norm(tensors):
    return torch.stack([t.float().square().sum() for t in tensors]).sum().sqrt()


def _plain_clip(tensors, max_norm):
    norm = _plain_norm(tensors)
    coef = (max_norm / (norm + NORM_EPS)).clamp(max=1.0)
    [t.copy_(t.float() * coef) for t in tensors]
    return norm


def _plain_adam(s):
    norm = _plain_norm(s['g'])
    coef = (s['max_norm'] / (norm + NORM_EPS)).clamp(max=1.0)
    s['t'] += 1
    grads = [g * coef + DECAY * p for g, p in zip(s['g'], s['p'])]
    s['m'] = [BETA1 * m + (1 - BETA1) * g for m, g in zip(s['m'], grads)]
    s['v'] = [BETA2 * v + (1 - BETA2) * g * g for v, g in zip(s['v'], grads)]
    if s['vmax'] is not None:
        s['vmax'] = [torch.maximum(x, v) for x, v in zip(s['vmax'], s['v'])]
    root = math.sqrt(1 - BETA2 ** s['t'])
    step = LR / (1 - BETA1 ** s['t'])
    s['p'] = [p - step * m / (v.sqrt() / root + EPS)
              for p, m, v in zip(s['p'], s['m'], s['vmax'] if s['vmax'] is not None else s['v'])]
    return norm


# ----------------------------------------------------------------------------------------------------------------
# what a pass cannot do without, and its result in 64 bits
# ----------------------------------------------------------------------------------------------------------------
def work(case):
    if case['op'] == 'linear':
        m, k, n, e = case['rows'], case['k'], case['n'], TYPES[case['dtype']].itemsize
        read = m * k + n * k + case['bias'] * n + case['residual'] * m * n
        if not case['train']:
            return dict(bytes=e * (read + m * n), flops=2 * m * n * k)
        return dict(bytes=e * (read + m * n + m * n + m * k + n * k + case['bias'] * n), flops=6 * m * n * k)
    if case['op'] == 'adam':
        return dict(bytes=4 * case['total'] * (9 if case['amsgrad'] else 7), flops=16 * case['total'])
    sizes = _sizes(case['count'], case['total'])
    half = {'fp32': 0, 'bf16': int(sizes.sum()), 'mixed': int(sizes[2::3].sum())}[case['dtype']]
    size = 4 * case['total'] - 2 * half
    return dict(bytes=size if case['op'] == 'norm' else 2 * size, flops=2 * case['total'])


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case['op'] == 'linear':
            return _exact_linear(s, case)
        if case['op'] == 'adam':
            return _exact_adam(s)
        total = torch.zeros((), device='cuda', dtype=torch.float64)
        for flat in s['flats']:                    # the padding between the tensors is zero
            for part in flat.split(1 << 26):
                total += part.double().pow(2).sum()
        norm = total.sqrt()
        if case['op'] == 'norm':
            return norm
        coef = min(1.0, s['max_norm'] * 0.999 / (float(norm) + NORM_EPS))
        return dict(norm=norm, grads=[f.double() * coef for f in s['flats']])


def _exact_linear(s, case):
    x, w = s['x'].double(), s['w'].double()
    z = (x @ w.t() + (0 if s['b'] is None else s['b'].double())).requires_grad_(True)
    fn = torch.nn.functional
    with torch.enable_grad():
        h = {'none': lambda v: v * 1.0, 'relu': fn.relu, 'leaky0.2': lambda v: fn.leaky_relu(v, 0.2),
             'tanh': torch.tanh, 'gelu': fn.gelu, 'gelu_tanh': lambda v: fn.gelu(v, approximate='tanh'),
             'silu': fn.silu}[case['act']](z)
    out = dict(y=h.detach() + (0 if s['r'] is None else s['r'].double()))
    if case['train']:
        dz, = torch.autograd.grad(h, z, s['gy'].double())
        out['dx'], out['dw'] = torch.mm(dz, w), torch.mm(dz.t().contiguous(), x)
        if s['b'] is not None:
            out['db'] = dz.sum(0)
        if s['r'] is not None:
            out['dr'] = s['gy'].double()
    return out


def _exact_adam(s):
    norm = math.sqrt(sum(float(g.double().pow(2).sum()) for g in s['g']))
    coef = min(1.0, s['max_norm'] / (norm + NORM_EPS))
    t = STEPS + 1
    out = dict(norm=torch.tensor(norm, dtype=torch.float64), p=[], m=[], v=[], vmax=[])
    for i, (p, g, m, v) in enumerate(zip(s['p'], s['g'], s['m'], s['v'])):
        p, g, m, v = (a.double() for a in (p, g, m, v))
        g = coef * g + DECAY * p
        m, v = m + (1.0 - BETA1) * (g - m), v + (1.0 - BETA2) * (g * g - v)
        x = v
        if s['vmax'] is not None:
            x = torch.maximum(s['vmax'][i].double(), v)
            out['vmax'].append(x)
        out['p'].append(p - LR * (m / (1.0 - BETA1 ** t)) / ((x / (1.0 - BETA2 ** t)).sqrt() + EPS))
        out['m'].append(m)
        out['v'].append(v)
    if s['vmax'] is None:
        del out['vmax']
    return out
