"""Plain 64-bit restatements of a gated recurrence block: the recurrence, the norms either side of the block, its projections; each with
its gradient written out.

As in head_oracle every function also returns the magnitudes that its results are made of, from which a test derives how far a 32-bit
computation of the same formulas may be off.
"""
import math

import torch

U = 2.0 ** -24   # half a step of fp32


def recurrence(x, g, h0, bounds, dh=None, dht=None):
    """x, g [rows, D] in their own type, h0 [n_seq, D] or None, token by token.  `<name>_off`: how far fp32 may be off.

    Per token: the decay (2 ulp = 4 U, its exponent |g| U), a product and a sum; the tokens of a step are joined by products
    of the decays and run through once more, which doubles that, and joining warps and steps adds a product and a sum each: 16 + 2 |g|
    in units of U times what is multiplied, with what was off before carried on by the same decays."""
    x, g = x.double(), g.double()
    a = torch.exp(g)
    unit = (16 + 2 * g.clamp(min=-200).abs()) * U
    D = x.shape[1]
    zero = x.new_zeros(D)
    out = {k: torch.zeros_like(x) for k in ('h', 'h_off')}
    out['ht'], out['ht_off'] = x.new_zeros(len(bounds), D), x.new_zeros(len(bounds), D)
    if dh is not None or dht is not None:
        dh = torch.zeros_like(x) if dh is None else dh.double()
        for k in ('dx', 'dx_off', 'dg', 'dg_off'):
            out[k] = torch.zeros_like(x)
        out['dh0'], out['dh0_off'] = x.new_zeros(len(bounds), D), x.new_zeros(len(bounds), D)
    for n, (lo, hi) in enumerate(bounds):
        h = zero if h0 is None else h0[n].double()
        size, off = h.abs(), zero
        before, before_off = [], []
        for t in range(lo, hi):
            before.append(h)
            before_off.append(off)
            carried = torch.where(a[t] > 0, a[t] * size, 0.0)
            off = torch.where(a[t] > 0, a[t] * off, 0.0) + unit[t] * (carried + x[t].abs())
            size = carried + x[t].abs()
            h = a[t] * h + x[t]
            out['h'][t], out['h_off'][t] = h, off
        out['ht'][n], out['ht_off'][n] = h, off
        if 'dx' not in out:
            continue
        u = zero if dht is None else dht[n].double()
        size, off = u.abs(), zero
        for t in range(hi - 1, lo - 1, -1):
            d = dh[t] + u
            size = size + dh[t].abs()
            off = off + unit[t] * size
            m = a[t] * before[t - lo]
            out['dx'][t], out['dx_off'][t] = d, off
            out['dg'][t] = d * m
            out['dg_off'][t] = m.abs() * off + (size + off) * (a[t] * before_off[t - lo] + unit[t] * m.abs())
            u, size, off = a[t] * d, a[t] * size, a[t] * off + unit[t] * a[t] * size
        out['dh0'][n], out['dh0_off'][n] = u, off
    return out


def dense_bounds(B, T):
    return [(b * T, (b + 1) * T) for b in range(B)]


def packed_bounds(cu):
    return list(zip(cu[:-1], cu[1:]))


def _activation(name, g):
    """The activation, its derivative, and the magnitudes that these are made of."""
    s = torch.sigmoid(g)
    if name == 'sigmoid':
        return s, s * (1 - s), s, s
    if name in ('silu', 'swish'):
        return g * s, s * (1 + g * (1 - s)), g.abs() * s, s * (1 + g.abs())
    if name == 'gelu':
        cdf = 0.5 * torch.special.erfc(-g * math.sqrt(0.5))
        pdf = torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
        return g * cdf, cdf + g * pdf, g.abs() * (cdf + 0.5), cdf + 0.5 + g.abs() * pdf
    return g, torch.ones_like(g), g.abs(), torch.ones_like(g)


def rms_norms(y, weight, residual, post, post_weight, gate, activation, scale, eps, dout=None, dz=None):
    """y, residual, gate [N, D] and parameters [D] (or None; scale may be a number) in their own types; `<name>_size` beside each result."""
    y = y.double()
    one = y.new_ones(y.shape[1])
    w = one if weight is None else weight.double()
    w1 = one if post_weight is None else post_weight.double()
    c = one if scale is None else scale.double() if isinstance(scale, torch.Tensor) else one * scale
    r1 = 1 / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) if post else torch.ones_like(y[:, :1])
    n1 = y * r1
    p = n1 * w1
    act, slope, act_size, slope_size = _activation(activation, gate.double()) if gate is not None else (torch.ones_like(y),) * 4
    res = torch.zeros_like(y) if residual is None else residual.double()
    z, z_size = res + c * act * p, res.abs() + (c * act_size * p).abs()
    r2 = 1 / torch.sqrt((z * z).mean(-1, keepdim=True) + eps)
    n2 = z * r2
    # an error of z by its size reaches r2 too
    carried = 1 + (z_size * z.abs()).mean(-1, keepdim=True) * r2 * r2
    n2_size = (z_size + z.abs() * carried) * r2
    out = {'z': z, 'z_size': z_size, 'out': n2 * w, 'out_size': n2_size * w.abs()}
    if dout is None and dz is None:
        return out
    dout = torch.zeros_like(y) if dout is None else dout.double()
    dz = torch.zeros_like(y) if dz is None else dz.double()
    h = dout * w
    e = dz + r2 * (h - n2 * (h * n2).mean(-1, keepdim=True))
    e_size = dz.abs() + r2 * carried * (h.abs() + n2_size * (h.abs() * n2_size).mean(-1, keepdim=True))
    f, f_size = e * c * act * w1, e_size * (c * act_size * w1).abs()
    dy, dy_size = (r1 * (f - n1 * (f * n1).mean(-1, keepdim=True)), r1 * (f_size + n1.abs() * (f_size * n1.abs()).mean(-1, keepdim=True))) if post else (f, f_size)
    out.update(dresidual=e, dresidual_size=e_size, dgate=e * c * p * slope, dgate_size=e_size * (c * p).abs() * slope_size, dy=dy, dy_size=dy_size,
               dweight=(dout * n2).sum(0), dweight_size=(dout.abs() * n2_size).sum(0),
               dpost_weight=(e * c * act * n1).sum(0), dpost_weight_size=(e_size * (c * act_size * n1).abs()).sum(0),
               dscale=(e * act * p).sum(0), dscale_size=(e_size * (act_size * p).abs()).sum(0))
    return out


def linear(x, weight, bias, residual, activation, dy=None):
    """x [M, K], weight [N, K], bias [N], residual [M, N] in their own 16-bit type; `<name>_off`: how far off fp32 sums may be.

    A sum of K products in steps of 16: (K / 16 + 32) units of 2^-23 of the sum of magnitudes.  The gradient reads z and dz rounded to the
    type (half a step each): the slope changes by at most 0.8 per unit of z."""
    half = torch.finfo(x.dtype).eps / 2

    def units(n):
        return (n / 16 + 32) * 2 * U
    x, w = x.double(), weight.double()
    b = w.new_zeros(w.shape[0]) if bias is None else bias.double()
    z, z_size = x @ w.t() + b, x.abs() @ w.abs().t() + b.abs()
    act, slope, act_size, slope_size = _activation(activation, z)
    z_off = units(x.shape[1]) * z_size
    y, y_off = act, 1.2 * z_off + (32 * U * act_size if activation else 0.0)
    if residual is not None:
        y, y_off = y + residual.double(), y_off + U * residual.double().abs()
    out = {'y': y, 'y_off': y_off}
    if dy is not None:
        dy = dy.double()
        dz = dy * slope
        unrounded = dy.abs() * (0.8 * (half * z.abs() + z_off) + 32 * U * slope_size) if activation else torch.zeros_like(dz)
        dz_off = unrounded + (half * dz.abs() if activation else 0.0)
        size = dz.abs() + dz_off
        out.update(dx=dz @ w, dx_off=dz_off @ w.abs() + units(w.shape[0]) * (size @ w.abs()),
                   dweight=dz.t() @ x, dweight_off=dz_off.t() @ x.abs() + units(x.shape[0]) * (size.t() @ x.abs()),
                   dbias=dz.sum(0), dbias_off=unrounded.sum(0) + units(x.shape[0]) * size.sum(0))
    return out
