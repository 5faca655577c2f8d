"""Plain 64-bit restatements of the steps around a stack of mixers: layer norm with its residual sum, log probabilities with
entropy and top alternatives, the divergence from a teacher's top entries; each with its gradient written out.

Every function also returns the magnitudes (sums of absolute values) that its results are made of, from which a test derives how far a
32-bit computation of the same formulas may be off.
"""
import math

import torch


def layer_norm(x, weight, bias, residual, eps, dy=None, dz=None):
    """x, residual [N, D] in their own type; returns a dict of 64-bit results."""
    z = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    zf = z.double()
    w = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if weight is None else weight.double()
    b = torch.zeros_like(w) if bias is None else bias.double()
    mean = zf.mean(-1, keepdim=True)
    c = zf - mean
    r = 1.0 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    n = c * r
    size = (zf.abs() + zf.abs().mean(-1, keepdim=True)) * r       # what n is the difference of
    out = {'z': z, 'y': n * w + b, 'y_size': size * w.abs() + b.abs()}
    if dy is not None:
        dy = dy.double()
        h = dy * w
        # sizes add up what goes into each term, and how far an error of n by `size` would carry
        reach = h.abs() + h.abs().mean(-1, keepdim=True) + size * (h.abs() * size).mean(-1, keepdim=True)
        out['dx'] = r * (h - h.mean(-1, keepdim=True) - n * (h * n).mean(-1, keepdim=True))
        out['dx_size'] = r * reach
        if dz is not None:
            out['dx'] = out['dx'] + dz.double()
            out['dx_size'] = out['dx_size'] + dz.double().abs()
        out['dweight'], out['dweight_size'] = (dy * n).sum(0), (dy.abs() * size).sum(0)
        out['dbias'], out['dbias_size'] = dy.sum(0), dy.abs().sum(0)
    return out


def _rows(x, temperature):
    """log probabilities, probabilities and which rows hold nothing but minus infinity (these have neither)"""
    x = x.double()
    top = x.amax(-1, keepdim=True)
    empty = top == -math.inf
    u = (x - torch.where(empty, 0.0, top)) / temperature
    e = torch.exp(u)
    s = e.sum(-1, keepdim=True)
    return torch.where(empty, -math.inf, u - torch.log(s)), torch.where(empty, 0.0, e / s), empty


def top_ids(x, k):
    """The k largest entries of each row, equal ones in the order of their indices (a stable sort keeps them so)."""
    return x.double().sort(dim=-1, descending=True, stable=True).indices[..., :k]


def logprobs(x, tokens, top_k, temperature, dlp=None, dh=None, dtop=None):
    """x [N, V]; returns a dict of 64-bit results and, where an upstream gradient is given, dx and dx_size."""
    lp, p, empty = _rows(x, temperature)
    given = (tokens >= 0) & (tokens < x.shape[-1])
    at = torch.where(given, tokens, 0).long()[:, None]
    given = given[:, None]
    plp = torch.where(p == 0, 0.0, p * lp)
    out = {'lp': lp, 'logprobs': torch.where(given, lp.gather(1, at), 0.0)[:, 0], 'entropy': 0.0 - plp.sum(-1)}
    if top_k:
        out['top_ids'] = top_ids(x, top_k)
        out['top_logprobs'] = lp.gather(1, out['top_ids'])
    if dlp is None and dh is None and dtop is None:
        return out
    zero = torch.zeros(x.shape[0], 1, dtype=torch.float64, device=x.device)
    dlp = zero if dlp is None else torch.where(given, dlp.double()[:, None], 0.0)
    dh = zero if dh is None else dh.double()[:, None]
    h = out['entropy'][:, None]
    all_of, all_size = dlp, dlp.abs()
    if dtop is not None:
        all_of, all_size = all_of + dtop.double().sum(-1, keepdim=True), all_size + dtop.double().abs().sum(-1, keepdim=True)
    dx = -(p * (all_of + dh * h) + dh * plp)
    size = p * (all_size + dh.abs() * h.abs()) + dh.abs() * plp.abs()
    dx.scatter_add_(1, at, dlp)
    size.scatter_add_(1, at, dlp.abs())
    if dtop is not None:
        dx.scatter_add_(1, out['top_ids'], dtop.double())
        size.scatter_add_(1, out['top_ids'], dtop.double().abs())
    out['dx'] = torch.where(empty, 0.0, dx / temperature)
    out['dx_size'] = torch.where(empty, 0.0, size / temperature)
    return out


REST_FROM = 1e-6   # less than this is what rounding leaves of a sum of one in 32 bits, and counts as nothing


def distill(x, teacher, ids, temperature, bucket):
    """x [N, V], teacher and ids [N, K]; per-row loss, which rows count, and the gradient of each row's loss."""
    lp, p, empty = _rows(x, temperature)
    V = x.shape[-1]
    there = (ids >= 0) & (ids < V) & ~(teacher.double() == -math.inf)
    at = torch.where(there, ids, 0).long()
    counted = there.any(-1)
    logq = torch.where(there, teacher.double(), -math.inf)
    if not bucket:
        logq = torch.where(counted[:, None], logq - torch.logsumexp(torch.where(counted[:, None], logq, 0.0), -1, keepdim=True), -math.inf)
    q = torch.where(there, logq.exp(), 0.0)
    given = lp.gather(1, at)
    term = torch.where(there & (q != 0), q * (torch.where(there, logq, 0.0) - given), 0.0)
    loss, size = term.sum(-1), torch.where(q != 0, q * (torch.where(there, logq, 0.0).abs() + given.abs()), 0.0).sum(-1)
    total = q.sum(-1, keepdim=True)
    listed = torch.zeros(x.shape, dtype=torch.int32, device=x.device).scatter_add_(1, at, there.int()) > 0
    rest = 1.0 - total if bucket else torch.zeros_like(total)
    rest = torch.where(rest < REST_FROM, 0.0, rest)
    share = p * (total + rest)
    reach = share.clone()
    if bucket:
        off = torch.where(listed, 0.0, p)
        p_rest = off.sum(-1, keepdim=True)
        some = rest[:, 0] > 0
        part = rest * (torch.log(rest) - torch.log(p_rest))
        loss = loss + torch.where(some, part[:, 0], 0.0)
        size = size + torch.where(some, (rest * (torch.log(rest).abs() + torch.log(p_rest).abs() + 2.0))[:, 0], 0.0)
        moved = torch.where(off == 0, 0.0, rest * off / torch.where(p_rest == 0, 1.0, p_rest))
        share = share - moved
        # the rest is one minus a sum in 32 bits: off by about an ulp of one, and so is its share of the gradient
        reach = reach + moved + torch.where(off == 0, 0.0, off / torch.where(p_rest == 0, 1.0, p_rest))
    dx = share.scatter_add(1, at, -q)
    reach = reach.scatter_add(1, at, q.abs())
    nothing = empty | ~counted[:, None]
    loss = torch.where(empty[:, 0] & counted, math.inf, loss)
    return {'rows': torch.where(counted, loss, 0.0), 'rows_size': torch.where(counted, size, 0.0), 'counted': counted,
            'dx': torch.where(nothing, 0.0, dx / temperature), 'dx_size': torch.where(nothing, 0.0, reach / temperature)}


def reduce_loss(rows, counted, reduction):
    """The reduced loss and the factor of each row's gradient in it."""
    if reduction == 'none':
        return rows, 1.0
    n = max(1, int(counted.sum())) if reduction == 'mean' else 1
    return rows.sum() / n, 1.0 / n
