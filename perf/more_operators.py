"""A gated recurrence block around the framework's mixers, as cases that can be timed and compared: the recurrence itself, the norms
either side of a block, the projections in and out of it.

A case names a path (`"path"`), its sizes and options:

* ``recurrence``  ``gated_recurrence``: ``h_t = exp(g_t) h_{t-1} + x_t`` a channel, for ``batch`` sequences of ``tokens`` tokens of ``dim``
                  channels, or (``packed`` > 0) one buffer of ``tokens`` that holds that many sequences; ``gate``: the type of g; ``state``:
                  there is an initial state, and the final one is handed back; with ``train`` the gradients of x, g and the initial state.
* ``norm``        ``residual_rms_norm``: ``rows`` rows of ``dim``: the norm of a block's output (``post``), its gate (``gate``: the
                  activation, or an empty text), its residual scale (``scale``), the residual sum, the norm ahead of the next block.
* ``linear``      ``fused_linear``: ``rows`` rows, ``inner`` to ``outer`` features, with bias, activation, residual; with ``train`` the
                  gradients of all of them.

Where ``own`` is false the operators are computed in elementary torch operations, in 32 bits, by the formulas.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
EPS = 1e-6
MOST_RECURRENT, MOST_NORM, MOST_LINEAR = 131072 * 1024, 65536 * 4096, 16384 * 2048 * 8192   # of the largest listed cases


def listed():
    return [
        # the recurrence in a decoding step of four users
        dict(name='recurrence_step_4x2048', path='recurrence', batch=4, tokens=1, dim=2048, packed=0, dtype='bf16', gate='bf16', state=True, train=False),
        # a training step of four sequences of 4096 tokens
        dict(name='recurrence_train_4x4096x2048', path='recurrence', batch=4, tokens=4096, dim=2048, packed=0, dtype='bf16', gate='bf16', state=False, train=True),
        # documents of any length packed into one buffer, an odd width, fp32
        dict(name='recurrence_train_packed_odd', path='recurrence', batch=1, tokens=8191, dim=1003, packed=13, dtype='fp32', gate='fp32', state=True, train=True),
        # the prompt of one user with a very long document, decays in fp32
        dict(name='recurrence_prompt_131072x1024', path='recurrence', batch=1, tokens=131072, dim=1024, packed=0, dtype='bf16', gate='fp32', state=True, train=False),
        # the norms between two blocks in a decoding step of four users
        dict(name='norms_step_4x2048', path='norm', rows=4, dim=2048, dtype='bf16', param='bf16', post=True, gate='', scale=True, residual=True, train=False),
        # a training step of four sequences of 4096 tokens, the block's output gated
        dict(name='norms_train_16384x2048', path='norm', rows=16384, dim=2048, dtype='bf16', param='fp32', post=True, gate='sigmoid', scale=True, residual=True, train=True),
        # an odd width in fp32
        dict(name='norms_train_odd_fp32', path='norm', rows=8191, dim=1003, dtype='fp32', param='fp32', post=True, gate='silu', scale=False, residual=True, train=True),
        # a wide model over a large training batch
        dict(name='norms_train_65536x4096', path='norm', rows=65536, dim=4096, dtype='bf16', param='bf16', post=True, gate='', scale=True, residual=True, train=True),
        # the projection into a block in a decoding step of four users
        dict(name='linear_step_4', path='linear', rows=4, inner=2048, outer=8192, dtype='bf16', bias=True, activation='silu', residual=False, train=False),
        # the projection back into the residual stream for a serving engine's batch
        dict(name='linear_step_200', path='linear', rows=200, inner=8192, outer=2048, dtype='bf16', bias=False, activation='', residual=True, train=False),
        # a short document, odd widths, fp16
        dict(name='linear_train_odd_fp16', path='linear', rows=1021, inner=1003, outer=2050, dtype='fp16', bias=True, activation='gelu', residual=True, train=True),
        # a training step of four sequences of 4096 tokens
        dict(name='linear_train_16384', path='linear', rows=16384, inner=2048, outer=8192, dtype='bf16', bias=True, activation='silu', residual=False, train=True),
    ]


def _log_int(rng, lo, hi):
    """An integer from [lo, hi], spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A width: more often than not a multiple of 64."""
    n = _log_int(rng, lo, hi)
    return max(lo, n // 64 * 64) if rng.random() < 0.65 else n


def draw(rng):
    path = rng.choice(['recurrence', 'norm', 'linear'])
    dtype = rng.choice(['bf16', 'bf16', 'fp16', 'fp32'])
    if path == 'recurrence':
        dim = _width(rng, 32, 8192)
        total = _log_int(rng, 1, min(131072, MOST_RECURRENT // (4 if dtype == 'fp32' else 2) // dim))
        case = dict(path=path, dim=dim, dtype=dtype, gate=rng.choice([dtype, dtype, 'fp32']), state=rng.random() < 0.6, train=rng.random() < 0.6)
        if rng.random() < 0.4:
            return dict(case, batch=1, tokens=total, packed=_log_int(rng, 1, max(1, min(256, total // 16))))
        batch = _log_int(rng, 1, min(64, total))
        return dict(case, batch=batch, tokens=max(1, total // batch), packed=0)
    if path == 'norm':
        dim = _width(rng, 64, 8192)
        return dict(path=path, rows=_log_int(rng, 1, min(65536, MOST_NORM // (4 if dtype == 'fp32' else 2) // dim)), dim=dim, dtype=dtype,
                    param=rng.choice([dtype, 'fp32']), post=rng.random() < 0.7, gate=rng.choice(['', '', 'sigmoid', 'silu']),
                    scale=rng.random() < 0.5, residual=rng.random() < 0.8, train=rng.random() < 0.6)
    inner, outer = _width(rng, 64, 8192), _width(rng, 64, 8192)
    rows = _log_int(rng, 1, min(32768, MOST_LINEAR // inner // outer))
    return dict(path=path, rows=rows, inner=inner, outer=outer, dtype='fp16' if dtype == 'fp16' else 'bf16', bias=rng.random() < 0.6,
                activation=rng.choice(['', '', 'silu', 'gelu', 'sigmoid']), residual=rng.random() < 0.4, train=rng.random() < 0.5)


class _Maker:
    def __init__(self, seed):
        self.dev = torch.device('cuda')
        self.gen = torch.Generator(device=self.dev).manual_seed(seed)
        self.rng = random.Random(seed)

    def normal(self, *shape, dtype=torch.float32, scale=1.0):
        return torch.empty(shape, dtype=torch.float32, device=self.dev).normal_(0.0, scale, generator=self.gen).to(dtype)

    def uniform(self, *shape):
        return torch.empty(shape, dtype=torch.float32, device=self.dev).uniform_(generator=self.gen)


def _lengths(m, total, n):
    """n sequences of one token at least, some much longer than others."""
    share = [m.rng.random() ** 2 + 0.02 for _ in range(n)]
    scale = (total - n) / sum(share)
    lens = [1 + int(s * scale) for s in share]
    lens[m.rng.randrange(n)] += total - sum(lens)
    return lens


def prepare(case, seed):
    m = _Maker(seed)
    dtype, train = DTYPES[case['dtype']], case['train']
    s = {'case': case}
    if case['path'] == 'recurrence':
        b, t, d = case['batch'], case['tokens'], case['dim']
        lens = _lengths(m, t, case['packed']) if case['packed'] else [t] * b
        s['starts'] = [sum(lens[:i]) for i in range(len(lens) + 1)]
        if case['packed']:
            s['cu_cpu'] = torch.tensor(s['starts'], dtype=torch.int32)
            s['cu'] = s['cu_cpu'].to(m.dev)
        # channels forget over one to a thousand tokens, each token a little differently
        slow = torch.exp(-7.0 * m.uniform(d))
        s['x'] = m.normal(b, t, d, dtype=dtype)
        s['g'] = (-slow * torch.nn.functional.softplus(m.normal(b, t, d) + 0.5)).to(DTYPES[case['gate']])
        s['h0'] = m.normal(len(lens), d, scale=2.0) if case['state'] else None
        s['leaves'] = [x for x in (s['x'], s['g'], s['h0']) if x is not None]
        if train:
            s['grads'] = [m.normal(b, t, d, dtype=dtype)] + ([m.normal(len(lens), d)] if case['state'] else [])
    elif case['path'] == 'norm':
        n, d, p = case['rows'], case['dim'], DTYPES[case['param']]
        # a block's output, not centred, beside a residual stream of larger spread
        s['y'] = (m.normal(n, d) + 0.3 * m.normal(1, d)).to(dtype)
        s['residual'] = (m.normal(n, d, scale=3.0) + m.normal(1, d)).to(dtype) if case['residual'] else None
        s['gate'] = m.normal(n, d, dtype=dtype) if case['gate'] else None
        s['weight'] = (1.0 + m.normal(d, scale=0.2)).to(p)
        s['post'] = (1.0 + m.normal(d, scale=0.2)).to(p) if case['post'] else None
        s['scale'] = (0.5 + m.normal(d, scale=0.1)).to(p) if case['scale'] else None
        s['names'] = [k for k in ('y', 'residual', 'gate', 'weight', 'post', 'scale') if s[k] is not None]
        s['leaves'] = [s[k] for k in s['names']]
        if train:
            s['grads'] = [m.normal(n, d, dtype=dtype), m.normal(n, d, dtype=dtype)]
    else:
        n, k, o = case['rows'], case['inner'], case['outer']
        s['x'] = m.normal(n, k, dtype=dtype)
        s['weight'] = m.normal(o, k, dtype=dtype, scale=k ** -0.5)
        s['bias'] = m.normal(o, dtype=dtype, scale=0.3) if case['bias'] else None
        s['residual'] = m.normal(n, o, dtype=dtype) if case['residual'] else None
        s['names'] = [k for k in ('x', 'weight', 'bias', 'residual') if s[k] is not None]
        s['leaves'] = [s[k] for k in s['names']]
        if train:
            s['grads'] = [m.normal(n, o, dtype=dtype)]
    for x in s['leaves']:
        x.requires_grad_(train)
    return s


# ---- the operators in elementary operations -----------------------------------------------------------------------
def _doubling(a, b):
    """h_t = a_t h_{t-1} + b_t along the second dimension, by steps that join twice as many tokens each."""
    step = 1
    while step < a.shape[1]:
        b = torch.cat([b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]], 1)
        a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], 1)
        step *= 2
    return b


def _sequences(s):
    """First and last token of every sequence as indices of [batch, tokens] flattened."""
    case = s['case']
    if case['packed']:
        first, last = s['starts'][:-1], [e - 1 for e in s['starts'][1:]]
    else:
        first = [i * case['tokens'] for i in range(case['batch'])]
        last = [i + case['tokens'] - 1 for i in first]
    dev = s['x'].device
    return torch.tensor(first, device=dev), torch.tensor(last, device=dev)


def _plain_recurrence(s):
    case = s['case']
    first, last = _sequences(s)
    x, a = s['x'].detach().float(), torch.exp(s['g'].detach().float())
    shape, d = x.shape, x.shape[-1]
    b, cut = x.reshape(-1, d).clone(), a.reshape(-1, d).clone()
    if case['state']:
        b[first] += cut[first] * s['h0'].detach()
    cut[first] = 0.0
    h = _doubling(cut.view(shape), b.view(shape))
    out = {'h': h.to(s['x'].dtype)}
    if case['state']:
        out['state'] = h.reshape(-1, d)[last]
    if case['train']:
        dh = s['grads'][0].float().reshape(-1, d).clone()
        if case['state']:
            dh[last] += s['grads'][1]
        # what reaches token t from t + 1 goes by the decay of t + 1, and nothing does across sequences
        after = torch.cat([cut[1:], torch.zeros_like(cut[:1])], 0).view(shape)
        dh = _doubling(after.flip(1), dh.view(shape).flip(1)).flip(1)
        before = torch.cat([torch.zeros_like(cut[:1]), h.reshape(-1, d)[:-1]], 0)
        before[first] = s['h0'].detach() if case['state'] else 0.0
        out['dx'] = dh.to(s['x'].dtype)
        out['dg'] = (dh * a * before.view(shape)).to(s['g'].dtype)
        if case['state']:
            out['dh0'] = (dh * a).reshape(-1, d)[first]
    return out


def _sigmoid(x):
    return 1.0 / (1.0 + torch.exp(-x))


def _activation(name, x):
    """The activation and its derivative."""
    if name == 'gelu':
        cdf = 0.5 * (1.0 + torch.erf(x * math.sqrt(0.5)))
        return x * cdf, cdf + x * torch.exp(-0.5 * x * x) * (1.0 / math.sqrt(2.0 * math.pi))
    if name == 'silu':
        e = _sigmoid(x)
        return x * e, e * (1.0 + x * (1.0 - e))
    if name == 'sigmoid':
        e = _sigmoid(x)
        return e, e * (1.0 - e)
    return x, torch.ones_like(x)


def _plain_norm(s):
    case = s['case']
    dtype = s['y'].dtype
    v = {k: s[k].detach().float() for k in s['names']}
    y = v['y']
    r1 = 1.0 / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS)
    n1 = y * r1 if case['post'] else y
    p = n1 * v['post'] if case['post'] else y
    act, slope = _activation(case['gate'], v['gate']) if case['gate'] else (1.0, None)
    scale = v['scale'] if case['scale'] else 1.0
    z = p * act * scale
    if case['residual']:
        z = z + v['residual']
    r2 = 1.0 / torch.sqrt((z * z).mean(-1, keepdim=True) + EPS)
    n2 = z * r2
    out = {'out': (n2 * v['weight']).to(dtype), 'z': z.to(dtype)}
    if case['train']:
        dout, dz = (g.float() for g in s['grads'])
        h = dout * v['weight']
        dz = dz + r2 * (h - n2 * (h * n2).mean(-1, keepdim=True))
        out['dweight'] = (dout * n2).sum(0).to(s['weight'].dtype)
        if case['residual']:
            out['dresidual'] = dz.to(dtype)
        if case['scale']:
            out['dscale'] = (dz * act * p).sum(0).to(s['scale'].dtype)
        if case['gate']:
            out['dgate'] = (dz * scale * p * slope).to(dtype)
        dp = dz * scale * act
        if case['post']:
            out['dpost'] = (dp * n1).sum(0).to(s['post'].dtype)
            h = dp * v['post']
            dp = r1 * (h - n1 * (h * n1).mean(-1, keepdim=True))
        out['dy'] = dp.to(dtype)
    return out


def _plain_linear(s):
    case = s['case']
    dtype = s['x'].dtype
    v = {k: s[k].detach().float() for k in s['names']}
    z = v['x'] @ v['weight'].t()
    if case['bias']:
        z = z + v['bias']
    y, slope = _activation(case['activation'], z)
    if case['residual']:
        y = y + v['residual']
    out = {'y': y.to(dtype)}
    if case['train']:
        dz = s['grads'][0].float() * slope
        out['dx'] = (dz @ v['weight']).to(dtype)
        out['dweight'] = (dz.t() @ v['x']).to(dtype)
        if case['bias']:
            out['dbias'] = dz.sum(0).to(dtype)
        if case['residual']:
            out['dresidual'] = s['grads'][0]
    return out


# ---- the framework's operators ------------------------------------------------------------------------------------
def _package():
    at = os.path.join(os.getcwd(), 'flash-linear-attention_b200')
    if at not in sys.path:
        sys.path.insert(0, at)
    import b200gdn
    return b200gdn


def _own_recurrence(s):
    case = s['case']
    h, state = _package().gated_recurrence(s['x'], s['g'], initial_state=s['h0'], output_final_state=case['state'],
                                           cu_seqlens=s.get('cu'), cu_seqlens_cpu=s.get('cu_cpu'))
    out = {'h': h.detach()}
    if case['state']:
        out['state'] = state.detach()
    if case['train']:
        out.update(zip(['dx', 'dg', 'dh0'], torch.autograd.grad([h] + ([state] if case['state'] else []), s['leaves'], s['grads'])))
    return out


def _own_norm(s):
    case = s['case']
    out, z = _package().residual_rms_norm(s['y'], s['weight'], residual=s['residual'], post_norm=case['post'], post_weight=s['post'],
                                          gate=s['gate'], gate_activation=case['gate'] or None, scale=s['scale'], eps=EPS)
    got = {'out': out.detach(), 'z': z.detach()}
    if case['train']:
        got.update(zip(['d' + k for k in s['names']], torch.autograd.grad([out, z], s['leaves'], s['grads'])))
    return got


def _own_linear(s):
    case = s['case']
    y = _package().fused_linear(s['x'], s['weight'], s['bias'], residual=s['residual'], activation=case['activation'] or None)
    out = {'y': y.detach()}
    if case['train']:
        out.update(zip(['d' + k for k in s['names']], torch.autograd.grad(y, s['leaves'], s['grads'])))
    return out


def run(state):
    path, train = state['case']['path'], state['case']['train']
    with torch.set_grad_enabled(own and train):
        if own:
            return {'recurrence': _own_recurrence, 'norm': _own_norm, 'linear': _own_linear}[path](state)
        return {'recurrence': _plain_recurrence, 'norm': _plain_norm, 'linear': _plain_linear}[path](state)


def work(case):
    """Bytes: each input read once, each output written once; what lies between a step's forward and backward pass is not
    counted.  Operations: a multiplication or an addition each, an exponential as one."""
    size, train = DTYPES[case['dtype']].itemsize, case['train']
    if case['path'] == 'recurrence':
        n, d = case['batch'] * case['tokens'], case['dim']
        gate = DTYPES[case['gate']].itemsize
        states = (case['packed'] or case['batch']) * d * 4 * (2 if case['state'] else 0) * (2 if train else 1)
        return {'bytes': n * d * (2 * size + gate + (2 * size + gate if train else 0)) + states, 'flops': n * d * (3 if not train else 9)}
    if case['path'] == 'norm':
        n, d = case['rows'], case['dim']
        read = 1 + case['residual'] + bool(case['gate'])
        params = d * DTYPES[case['param']].itemsize * (1 + case['post'] + case['scale']) * (2 if train else 1)
        return {'bytes': n * d * size * (read + 2 + (2 + read if train else 0)) + params, 'flops': n * d * (14 if not train else 46)}
    n, k, o = case['rows'], case['inner'], case['outer']
    tensors = n * k + o * k + case['bias'] * o
    return {'bytes': size * ((tensors + case['residual'] * n * o) * (2 if train else 1) + n * o * (2 if train else 1)),
            'flops': 2 * n * k * o * (3 if train else 1)}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case['path'] == 'recurrence':
        return _exact_recurrence(s)
    with torch.enable_grad():
        return {'norm': _exact_norm, 'linear': _exact_linear}[case['path']](s)


def _exact_scan(a, b, h):
    """h_t = a_t h_{t-1} + b_t along the first dimension, from h: 64 tokens side by side in blocks, then block after block."""
    t, d = a.shape
    n = -(-t // 64)
    pad = n * 64 - t
    a = torch.cat([a, a.new_ones(pad, d)]).view(n, 64, d)
    b = torch.cat([b, b.new_zeros(pad, d)]).view(n, 64, d)
    inside, through = torch.empty_like(b), torch.empty_like(a)
    e, p = torch.zeros_like(b[:, 0]), torch.ones_like(a[:, 0])
    for i in range(64):
        e = a[:, i] * e + b[:, i]
        p = a[:, i] * p
        inside[:, i], through[:, i] = e, p
    entering = torch.empty_like(e)
    for j in range(n):
        entering[j] = h
        h = inside[j, -1] + through[j, -1] * h
    return (inside + through * entering[:, None]).view(-1, d)[:t]


def _exact_recurrence(s):
    case = s['case']
    d = case['dim']
    x, g = (s[k].detach().double().view(-1, d) for k in ('x', 'g'))
    a = torch.exp(g)
    bounds = [(i * case['tokens'], (i + 1) * case['tokens']) for i in range(case['batch'])]
    if case['packed']:
        bounds = list(zip(s['starts'][:-1], s['starts'][1:]))
    names = ['h'] + (['state'] if case['state'] else []) + ((['dx', 'dg'] + (['dh0'] if case['state'] else [])) if case['train'] else [])
    out = {k: torch.empty_like(x) if k in ('h', 'dx', 'dg') else x.new_empty(len(bounds), d) for k in names}
    zero = x.new_zeros(d)
    for i, (lo, hi) in enumerate(bounds):
        h0 = s['h0'][i].detach().double() if case['state'] else zero
        h = _exact_scan(a[lo:hi], x[lo:hi], h0)
        out['h'][lo:hi] = h
        if case['state']:
            out['state'][i] = h[-1]
        if case['train']:
            from_after = torch.cat([a[lo + 1:hi], torch.ones_like(a[:1])])
            up = s['grads'][0].double().view(-1, d)[lo:hi]
            last = s['grads'][1][i].double() if case['state'] else zero
            dh = _exact_scan(from_after.flip(0), up.flip(0), last).flip(0)
            out['dx'][lo:hi] = dh
            out['dg'][lo:hi] = dh * a[lo:hi] * torch.cat([h0[None], h[:-1]])
            if case['state']:
                out['dh0'][i] = dh[0] * a[lo]
    return {k: v.view(s['x'].shape) if k in ('h', 'dx', 'dg') else v for k, v in out.items()}


def _exact_activation(name, x):
    return {'': lambda v: v, 'silu': lambda v: v * torch.sigmoid(v), 'sigmoid': torch.sigmoid,
            'gelu': lambda v: 0.5 * v * torch.special.erfc(-v / math.sqrt(2.0))}[name](x)


def _exact_norm(s):
    case = s['case']
    v = {k: s[k].detach().double().requires_grad_(case['train']) for k in s['names']}
    part = v['y']
    if case['post']:
        part = part / torch.sqrt(part.square().mean(-1, keepdim=True) + EPS) * v['post']
    if case['gate']:
        part = part * _exact_activation(case['gate'], v['gate'])
    if case['scale']:
        part = part * v['scale']
    z = part + v['residual'] if case['residual'] else part
    out = z / torch.sqrt(z.square().mean(-1, keepdim=True) + EPS) * v['weight']
    got = {'out': out.detach(), 'z': z.detach()}
    if case['train']:
        got.update(zip(['d' + k for k in s['names']], torch.autograd.grad([out, z], [v[k] for k in s['names']], [g.double() for g in s['grads']])))
    return got


def _exact_linear(s):
    case = s['case']
    v = {k: s[k].detach().double().requires_grad_(case['train']) for k in s['names']}
    y = _exact_activation(case['activation'], torch.nn.functional.linear(v['x'], v['weight'], v.get('bias')))
    if case['residual']:
        y = y + v['residual']
    out = {'y': y.detach()}
    if case['train']:
        out.update(zip(['d' + k for k in s['names']], torch.autograd.grad(y, [v[k] for k in s['names']], s['grads'][0].double())))
    return out


if __name__ == '__main__':
    for c in listed() + [draw(random.Random(i)) for i in range(8)]:
        print(c, work(c))
