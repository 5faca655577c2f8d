"""The steps around a stack of Gated DeltaNet mixers, as cases that can be timed and compared: the layer norm ahead of each
mixer and of the head, and what is done with the head's logits.

A case names a path (`"path"`), its sizes and options:

* ``norm``      ``layer_norm``: ``rows`` rows of ``dim``, with the residual sum (``residual``: the sum is handed on as well),
                with or without a bias, forward only or with its backward pass (``train``).
* ``logprobs``  ``token_logprobs``: ``rows`` rows of logits over ``vocab`` entries: the log probability of a given token a row, the
                entropy, the ``top`` most probable entries; with ``train`` the gradient of the logits, for upstream gradients of all
                of them.  ``masked``: a share of the entries is minus infinity, and a row here and there has nothing else.
* ``distill``   ``topk_distill_loss``: the student's logits against a teacher's ``top`` entries a row, mean over the rows that have
                any; with ``train`` the gradient of the logits.  ``bucket``: what the teacher leaves to the rest of the
                vocabulary counts as one more entry.

Where ``own`` is false the operators are computed in elementary torch operations, in 32 bits, by the formulas.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
EPS = 1e-5
MOST = 4096 * 131072      # logits of the largest listed case


def listed():
    return [
        # the norm ahead of a mixer in a decoding step of four users
        dict(name='norm_step_4x2048', path='norm', rows=4, dim=2048, dtype='bf16', param='bf16', residual=True, bias=True, train=False),
        # the same in a training step of four sequences of 4096 tokens
        dict(name='norm_train_16384x2048', path='norm', rows=16384, dim=2048, dtype='bf16', param='fp32', residual=True, bias=True, train=True),
        # rows of an odd width, in fp32, a sequence that is one token short
        dict(name='norm_train_odd_fp32', path='norm', rows=8191, dim=1003, dtype='fp32', param='fp32', residual=False, bias=False, train=True),
        # a wide model's norm over a large training batch
        dict(name='norm_train_65536x4096', path='norm', rows=65536, dim=4096, dtype='bf16', param='bf16', residual=False, bias=True, train=True),
        # one user's next token, with the alternatives that a completion interface shows
        dict(name='logprobs_step_1', path='logprobs', rows=1, vocab=131072, dtype='bf16', top=20, temperature=1.0, masked=False, train=False),
        # a serving engine's batch in fp32, constrained decoding
        dict(name='logprobs_step_256', path='logprobs', rows=256, vocab=32000, dtype='fp32', top=5, temperature=0.7, masked=True, train=False),
        # a teacher's pass over a prompt: its top entries are what a student learns from
        dict(name='logprobs_teacher_2048', path='logprobs', rows=2048, vocab=131072, dtype='bf16', top=64, temperature=1.0, masked=False, train=False),
        # a policy's step: log probabilities of the sampled tokens and an entropy bonus
        dict(name='logprobs_train_4096', path='logprobs', rows=4096, vocab=131072, dtype='bf16', top=0, temperature=1.0, masked=False, train=True),
        # an odd vocabulary in fp16, a penalty on the alternatives as well
        dict(name='logprobs_train_odd_fp16', path='logprobs', rows=1021, vocab=50001, dtype='fp16', top=8, temperature=1.3, masked=True, train=True),
        # a short document of a small student
        dict(name='distill_train_37', path='distill', rows=37, vocab=32000, dtype='bf16', top=20, temperature=1.0, bucket=False, train=True),
        # a student's training step
        dict(name='distill_train_4096', path='distill', rows=4096, vocab=131072, dtype='bf16', top=64, temperature=1.0, bucket=False, train=True),
        # an odd vocabulary in fp32, softened, with the rest of the vocabulary as an entry
        dict(name='distill_bucket_odd_fp32', path='distill', rows=2047, vocab=50001, dtype='fp32', top=32, temperature=2.0, bucket=True, train=True),
    ]


def _log_int(rng, lo, hi):
    """An integer from [lo, hi], spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    path = rng.choice(['norm', 'logprobs', 'distill'])
    dtype = rng.choice(['bf16', 'bf16', 'fp16', 'fp32'])
    if path == 'norm':
        dim = _log_int(rng, 64, 8192)
        if rng.random() < 0.6:
            dim = max(64, dim // 64 * 64)
        return dict(path=path, rows=_log_int(rng, 1, min(65536, 2 ** 27 // dim)), dim=dim, dtype=dtype, param=rng.choice([dtype, 'fp32']),
                    residual=rng.random() < 0.5, bias=rng.random() < 0.7, train=rng.random() < 0.6)
    if path == 'distill' and dtype == 'fp16':   # gradients of a mean over thousands of rows are below what fp16 holds
        dtype = 'bf16'
    vocab = _log_int(rng, 1000, 262144)
    if rng.random() < 0.5:
        vocab = max(1000, vocab // 64 * 64)
    rows = _log_int(rng, 1, min(32768, MOST // (4 if dtype == 'fp32' else 2) // vocab))
    common = dict(path=path, rows=rows, vocab=vocab, dtype=dtype, temperature=rng.choice([1.0, 1.0, 0.6, 2.0]))
    if path == 'logprobs':
        return dict(common, top=rng.choice([0, 1, 5, 20, 64, 128]), masked=rng.random() < 0.3, train=rng.random() < 0.5)
    return dict(common, top=_log_int(rng, 1, 128), bucket=rng.random() < 0.5, train=rng.random() < 0.75)


class _Maker:
    def __init__(self, seed):
        self.dev = torch.device('cuda')
        self.gen = torch.Generator(device=self.dev).manual_seed(seed)

    def normal(self, *shape, dtype=torch.float32, scale=1.0):
        return torch.empty(shape, dtype=torch.float32, device=self.dev).normal_(0.0, scale, generator=self.gen).to(dtype)

    def uniform(self, *shape):
        return torch.empty(shape, dtype=torch.float32, device=self.dev).uniform_(generator=self.gen)

    def below(self, n, *shape):
        return torch.randint(0, n, shape, device=self.dev, generator=self.gen)

    def distinct(self, rows, k, n):
        """k distinct entries of range(n) a row, in no order: sums of steps of at least one."""
        steps = 1 + (self.uniform(rows, k) * (n // k)).long().clamp(0, n // k - 1)
        ids = steps.cumsum(-1) - 1
        return ids.gather(-1, self.uniform(rows, k).argsort(-1))


def prepare(case, seed):
    m = _Maker(seed)
    dtype, n = DTYPES[case['dtype']], case['rows']
    s = {'case': case}
    if case['path'] == 'norm':
        d, p = case['dim'], DTYPES[case['param']]
        # a residual stream: of larger spread than what a block adds to it, not centred
        s['x'] = (m.normal(n, d) + 0.3 * m.normal(1, d)).to(dtype)
        s['residual'] = (m.normal(n, d, scale=3.0) + m.normal(1, d)).to(dtype) if case['residual'] else None
        s['weight'] = (1.0 + m.normal(d, scale=0.2)).to(p)
        s['bias'] = m.normal(d, dtype=p, scale=0.2) if case['bias'] else None
        s['leaves'] = [x for x in (s['x'], s['residual'], s['weight'], s['bias']) if x is not None]
        if case['train']:
            s['grads'] = [m.normal(n, d, dtype=dtype)] + ([m.normal(n, d, dtype=dtype)] if case['residual'] else [])
            for x in s['leaves']:
                x.requires_grad_(True)
        return s
    v, k = case['vocab'], case['top']
    # a head's logits: a broad floor with, in most rows, some entries well above it
    x = m.normal(n, v, scale=2.0)
    if case['path'] == 'logprobs':
        tokens = m.below(v, n)
        x.scatter_add_(1, tokens[:, None], 8.0 * m.uniform(n, 1))
        if case['masked']:
            x.masked_fill_(m.uniform(n, v) < 0.1, -math.inf)
            x[5::16] = -math.inf
        # prompts and padding: nothing is asked of these rows' tokens
        s['tokens'] = torch.where(m.uniform(n) < (0.2 if n > 8 else 0.0), -100, tokens)
        if case['train']:
            s['grads'] = [m.normal(n), m.normal(n, scale=0.1)] + ([m.normal(n, k, scale=0.3)] if k else [])
    else:
        ids = m.distinct(n, k, v)
        x.scatter_add_(1, ids, 4.0 + 2.0 * m.normal(n, k))
        # the teacher's log probabilities, most probable first; a few per cent are left to the rest of the vocabulary
        z = m.normal(n, k, scale=2.0).sort(-1, descending=True).values
        rest = z[:, :1] - 3.5 + 0.5 * m.normal(n, 1)
        s['teacher'] = z - torch.cat([z, rest], -1).logsumexp(-1, keepdim=True)
        if k > 4:   # some lists are shorter than others
            ids = torch.where((m.uniform(n, 1) < 0.2) & (torch.arange(k, device=m.dev) >= k - k // 4), -1, ids)
        if n > 8:   # rows of the prompt have no teacher
            ids = torch.where(m.uniform(n, 1) < 0.1, -1, ids)
        s['ids'] = ids
    s['logits'] = x.to(dtype).requires_grad_(case['train'])
    return s


# ---- the operators in elementary operations -----------------------------------------------------------------------
def _plain_norm(s):
    case = s['case']
    dtype = s['x'].dtype
    x, w = s['x'].detach(), s['weight'].detach().float()
    # what is handed on is rounded to its type, and normalised as the rest of the model will see it
    z = (x.float() + s['residual'].detach().float()).to(dtype) if case['residual'] else x
    zf = z.float()
    c = zf - zf.mean(-1, keepdim=True)
    r = 1.0 / torch.sqrt((c * c).mean(-1, keepdim=True) + EPS)
    n = c * r
    y = n * w
    if case['bias']:
        y = y + s['bias'].detach().float()
    out = {'y': y.to(dtype)}
    if case['residual']:
        out['z'] = z
    if case['train']:
        dy = s['grads'][0].float()
        h = dy * w
        dx = r * (h - h.mean(-1, keepdim=True) - n * (h * n).mean(-1, keepdim=True))
        if case['residual']:
            dx = dx + s['grads'][1].float()
        out['dx'] = dx.to(dtype)
        if case['residual']:
            out['dresidual'] = out['dx']
        out['dweight'] = (dy * n).sum(0).to(s['weight'].dtype)
        if case['bias']:
            out['dbias'] = dy.sum(0).to(s['bias'].dtype)
    return out


def _plain_rows(x, c):
    """Log probabilities and probabilities of rows of logits; a row that holds nothing but minus infinity has neither."""
    top = x.amax(-1, keepdim=True)
    empty = top == -math.inf
    u = (x - torch.where(empty, 0.0, top)) * c
    e = torch.exp(u)
    total = e.sum(-1, keepdim=True)
    lp = torch.where(empty, -math.inf, u - torch.log(total))
    return lp, torch.where(empty, 0.0, e / total), empty


def _plain_top(x, k):
    """The k largest entries of each row, ties to the lowest index: by keys of 64 bits that have no ties."""
    bits = (x + 0.0).view(torch.int32)
    value = torch.where(bits < 0, bits ^ 0x7fffffff, bits).long()
    last = x.shape[-1] - 1
    keys = (value << 32) | (last - torch.arange(x.shape[-1], device=x.device))
    return last - (keys.topk(k, dim=-1).values & 0xffffffff)


def _plain_logprobs(s):
    case = s['case']
    k, c = case['top'], 1.0 / case['temperature']
    x = s['logits'].detach().float()
    lp, p, empty = _plain_rows(x, c)
    plp = torch.where(p > 0, p * lp, 0.0)
    given = (s['tokens'] >= 0)[:, None]
    at = s['tokens'].clamp(min=0)[:, None]
    out = {'logprobs': torch.where(given, lp.gather(1, at), 0.0)[:, 0], 'entropy': -plp.sum(-1)}
    if k:
        out['top_ids'] = _plain_top(x, k)
        out['top_logprobs'] = lp.gather(1, out['top_ids'])
    if case['train']:
        d_lp = torch.where(given, s['grads'][0][:, None], 0.0)
        d_h, h = s['grads'][1][:, None], out['entropy'][:, None]
        all_of = d_lp + (s['grads'][2].sum(-1, keepdim=True) if k else 0.0)
        dx = -(p * (all_of + d_h * h) + d_h * plp)
        dx.scatter_add_(1, at, d_lp)
        if k:
            dx.scatter_add_(1, out['top_ids'], s['grads'][2])
        out['dlogits'] = torch.where(empty, 0.0, dx * c).to(s['logits'].dtype)
    return out


def _plain_distill(s):
    case = s['case']
    c = 1.0 / case['temperature']
    lp, p, _ = _plain_rows(s['logits'].detach().float(), c)
    there = s['ids'] >= 0
    ids = s['ids'].clamp(min=0)
    q = torch.where(there, torch.exp(s['teacher']), 0.0)
    counted = there.any(-1, keepdim=True)
    if not case['bucket']:
        q = q / torch.where(counted, q.sum(-1, keepdim=True), 1.0)
    log_q = torch.where(q > 0, torch.log(q), 0.0)
    loss = torch.where(q > 0, q * (log_q - lp.gather(1, ids)), 0.0).sum(-1, keepdim=True)
    on_list = torch.zeros_like(p, dtype=torch.int32).scatter_add_(1, ids, there.int()) > 0 if case['bucket'] else None
    share = p
    if case['bucket']:
        q_rest = (1.0 - q.sum(-1, keepdim=True)).clamp(min=0.0)
        p_rest = torch.where(on_list, 0.0, p).sum(-1, keepdim=True)
        loss = loss + torch.where(q_rest > 0, q_rest * (torch.log(q_rest) - torch.log(p_rest)), 0.0)
        share = p * (q.sum(-1, keepdim=True) + q_rest) - torch.where(on_list, 0.0, p / p_rest * q_rest)
    rows = counted.sum().clamp(min=1)
    out = {'loss': torch.where(counted, loss, 0.0).sum() / rows}
    if case['train']:
        dx = torch.scatter_add(share, 1, ids, -q)
        out['dlogits'] = (torch.where(counted, dx, 0.0) * (c / rows)).to(s['logits'].dtype)
    return out


# ---- the framework's operators ------------------------------------------------------------------------------------
def _package():
    at = os.path.join(os.getcwd(), 'flash-linear-attention_b200')
    if at not in sys.path:
        sys.path.insert(0, at)
    import b200gdn
    return b200gdn


def _own_norm(s):
    case = s['case']
    out = _package().layer_norm(s['x'], s['weight'], s['bias'], residual=s['residual'], eps=EPS, prenorm=case['residual'])
    names = ['y', 'z'] if case['residual'] else ['y']
    values = list(out) if case['residual'] else [out]
    got = dict(zip(names, (v.detach() for v in values)))
    if case['train']:
        got.update(zip(['dx'] + (['dresidual'] if case['residual'] else []) + ['dweight'] + (['dbias'] if case['bias'] else []),
                       torch.autograd.grad(values, s['leaves'], s['grads'])))
    return got


def _own_logprobs(s):
    case = s['case']
    r = _package().token_logprobs(s['logits'], s['tokens'], top_k=case['top'], temperature=case['temperature'])
    out = {'logprobs': r.logprobs.detach(), 'entropy': r.entropy.detach()}
    values = [r.logprobs, r.entropy]
    if case['top']:
        out.update(top_ids=r.top_ids, top_logprobs=r.top_logprobs.detach())
        values.append(r.top_logprobs)
    if case['train']:
        out['dlogits'], = torch.autograd.grad(values, s['logits'], s['grads'])
    return out


def _own_distill(s):
    case = s['case']
    loss = _package().topk_distill_loss(s['logits'], s['teacher'], s['ids'], temperature=case['temperature'],
                                        remainder='bucket' if case['bucket'] else 'renormalize')
    out = {'loss': loss.detach()}
    if case['train']:
        out['dlogits'], = torch.autograd.grad(loss, s['logits'])
    return out


def run(state):
    path, train = state['case']['path'], state['case']['train']
    with torch.set_grad_enabled(own and train):
        if own:
            return {'norm': _own_norm, 'logprobs': _own_logprobs, 'distill': _own_distill}[path](state)
        return {'norm': _plain_norm, 'logprobs': _plain_logprobs, 'distill': _plain_distill}[path](state)


def work(case):
    """Bytes: each input read once, each output written once; what lies between a step's forward and backward pass is not
    counted.  Operations: a multiplication or an addition each, an exponential as one."""
    n, size, grad = case['rows'], DTYPES[case['dtype']].itemsize, 2 if case['train'] else 1
    if case['path'] == 'norm':
        d, streams = case['dim'], 4 if case['residual'] else 2
        tensors = streams + (0 if not case['train'] else streams - (1 if case['residual'] else 0))   # dx serves both leaves
        params = d * DTYPES[case['param']].itemsize * (2 if case['bias'] else 1) * grad
        return {'bytes': n * d * size * tensors + params, 'flops': n * d * (8 if not case['train'] else 22)}
    v, k = case['vocab'], case['top']
    each = 8 + 8 + (16 if case['train'] else 0) if case['path'] == 'logprobs' else 0
    lists = k * (8 + 4 + (4 if case['train'] and case['path'] == 'logprobs' else 0))
    return {'bytes': n * v * size * grad + n * (each + lists), 'flops': n * v * (6 if not case['train'] else 14)}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.enable_grad():
        return {'norm': _exact_norm, 'logprobs': _exact_logprobs, 'distill': _exact_distill}[case['path']](s)


def _exact_norm(s):
    case = s['case']
    x = s['x'].detach()
    z = (x.double() + s['residual'].detach().double()).float().to(x.dtype) if case['residual'] else x
    z64, w = z.double().requires_grad_(True), s['weight'].detach().double().requires_grad_(True)
    leaves = [z64, w]
    if case['bias']:
        leaves.append(s['bias'].detach().double().requires_grad_(True))
    spread = torch.sqrt(z64.var(-1, keepdim=True, correction=0) + EPS)
    y = (z64 - z64.mean(-1, keepdim=True)) / spread * w + (leaves[2] if case['bias'] else 0.0)
    out = {'y': y.detach()}
    if case['residual']:
        out['z'] = z.double()
    if case['train']:
        d = torch.autograd.grad(y, leaves, s['grads'][0].double())
        out['dx'] = d[0] + (s['grads'][1].double() if case['residual'] else 0.0)
        if case['residual']:
            out['dresidual'] = out['dx']
        out['dweight'] = d[1]
        if case['bias']:
            out['dbias'] = d[2]
    return out


def _exact_logprobs(s):
    case = s['case']
    empty = (s['logits'].detach() == -math.inf).all(-1, keepdim=True)
    x = torch.where(empty, 0.0, s['logits'].detach().double()).requires_grad_(case['train'])
    lp = torch.log_softmax(x / case['temperature'], -1)
    given = s['tokens'] >= 0
    at = s['tokens'].clamp(min=0)[:, None]
    # minus infinity in a product with a probability of zero: its share of the entropy is nothing
    finite = torch.where(lp == -math.inf, 0.0, lp)
    chosen = torch.where(given, lp.gather(1, at)[:, 0], 0.0)
    entropy = -(finite.exp() * finite * (lp != -math.inf)).sum(-1)
    out = {'logprobs': torch.where(given & empty[:, 0], -math.inf, chosen.detach()), 'entropy': torch.where(empty[:, 0], 0.0, entropy.detach())}
    values = [chosen, entropy]
    if case['top']:
        top = lp.topk(case['top'], -1).values
        out['top_ids'], out['top_logprobs'] = None, torch.where(empty, -math.inf, top.detach())
        if case['train']:   # of entries with the same value the one with the lowest index has the gradient
            top = lp.gather(1, lp.detach().sort(dim=-1, descending=True, stable=True).indices[:, :case['top']])
        values.append(top)
    if case['train']:
        dx, = torch.autograd.grad(values, x, [g.double() for g in s['grads']])
        out['dlogits'] = torch.where(empty, 0.0, dx)
    return out


def _exact_distill(s):
    case = s['case']
    x = s['logits'].detach().double().requires_grad_(case['train'])
    lp = torch.log_softmax(x / case['temperature'], -1)
    there = s['ids'] >= 0
    ids = s['ids'].clamp(min=0)
    counted = there.any(-1)
    logq = torch.where(there, s['teacher'].double(), -math.inf)
    if not case['bucket']:
        logq = torch.where(there, torch.log_softmax(torch.where(counted[:, None], logq, 0.0), -1), -math.inf)
    q = logq.exp()
    rows = (q * (torch.where(there, logq, 0.0) - lp.gather(1, ids))).sum(-1)
    if case['bucket']:
        q_rest = (1.0 - q.sum(-1)).clamp(min=0.0)
        listed_ids = torch.zeros_like(lp, dtype=torch.int32).scatter_add_(1, ids, there.int())
        rest = torch.logsumexp(torch.where(listed_ids > 0, -math.inf, lp), -1)
        rows = rows + torch.where(q_rest > 0, q_rest * (torch.log(q_rest) - rest), 0.0)
    loss = torch.where(counted, rows, 0.0).sum() / counted.sum().clamp(min=1)
    out = {'loss': loss.detach()}
    if case['train']:
        out['dlogits'], = torch.autograd.grad(loss, x)
    return out


if __name__ == '__main__':
    for c in listed() + [draw(random.Random(i)) for i in range(8)]:
        print(c, work(c))
