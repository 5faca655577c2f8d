"""The RMS norms either side of a block on the GPU against the 64-bit restatement.

Tolerances: a result is rounded once to its type (half a step of the type, allowed twice: bf16 2^-8, fp16 2^-11, fp32 2^-24 relative), and
what is computed in 32 bits before may be off by a few units (2^-24) of the magnitudes it is made of: up to ten products and approximated
functions of a few units each, and sums over a row in chains of at most some tens of terms, for which 64 units are allowed in all."""
import ctypes as C
import itertools

import pytest
import torch

from oracle import block_oracle as O

pytestmark = pytest.mark.gpu
BF, HF, F = torch.bfloat16, torch.float16, torch.float32
EPS = {BF: 2.0 ** -8, HF: 2.0 ** -11, F: 2.0 ** -24}
TINY = {BF: 1e-37, HF: 2.0 ** -24, F: 1e-37}
UNITS = 64 * 2.0 ** -24


def close(name, got, want, size):
    limit = EPS[got.dtype] * want.abs() + UNITS * size + TINY[got.dtype]
    assert torch.isfinite(got).all(), name
    if got.numel():
        far = ((got.double() - want).abs() / limit).max().item()
        assert far <= 1.0, f'{name}: {far:.2f} of what is allowed'


def make(rows, D, dtype, ptype, seed=0):
    gen = torch.Generator(device='cuda').manual_seed(seed)

    def rn(*s):
        return torch.randn(*s, device='cuda', generator=gen)
    t = dict(y=(rn(rows, D) + 0.3).to(dtype), residual=(3 * rn(rows, D)).to(dtype), gate=(2 * rn(rows, D)).to(dtype),
             weight=(1 + 0.3 * rn(D)).to(ptype), post_weight=(1 + 0.3 * rn(D)).to(ptype), scale=(0.5 + 0.2 * rn(D)).to(ptype))
    return t, rn(rows, D).to(dtype), rn(rows, D).to(dtype)


NAMES = ('y', 'weight', 'residual', 'post_weight', 'gate', 'scale')


def call(t, post, activation, eps=1e-6):
    from b200gdn import residual_rms_norm
    return residual_rms_norm(t['y'], t.get('weight'), t.get('residual'), post, t.get('post_weight'), t.get('gate'), activation, t.get('scale'), eps)


def run_and_check(t, dout, dz, post, activation, eps=1e-6, upstream=('out', 'z')):
    leaves = {k: v.detach().clone().requires_grad_(True) if isinstance(v, torch.Tensor) else v for k, v in t.items()}
    out, z = call(leaves, post, activation, eps)
    use = [(o, g) for n, o, g in (('out', out, dout), ('z', z, dz)) if n in upstream]
    names = [k for k in NAMES if isinstance(leaves.get(k), torch.Tensor)]
    got = dict(zip(names, torch.autograd.grad([o for o, _ in use], [leaves[k] for k in names], [g for _, g in use])))
    want = O.rms_norms(t['y'], t.get('weight'), t.get('residual'), post, t.get('post_weight'), t.get('gate'), activation, t.get('scale'), eps,
                       dout if 'out' in upstream else None, dz if 'z' in upstream else None)
    close('out', out.detach(), want['out'], want['out_size'])
    close('z', z.detach(), want['z'], want['z_size'])
    for k, v in got.items():
        assert v.dtype == t[k].dtype
        close('d' + k, v, want['d' + k], want['d' + k + '_size'])
    with torch.no_grad():
        again = call(t, post, activation, eps)
    assert torch.equal(again[0], out) and torch.equal(again[1], z)


# what of the step is there: residual, post norm (its weight), gate (its activation), scale, weight
FORMS = [dict(residual=1, post=1, post_weight=1, gate='sigmoid', scale=1, weight=1), dict(residual=1, post=0, weight=1), dict(weight=1, post=0),
         dict(residual=1, post=1, gate='silu', weight=1), dict(post=1, post_weight=1, gate='', scale=1), dict(residual=1, post=0, gate='', scale=0.25, weight=1)]
WIDTHS = [1, 2, 7, 8, 33, 64, 100, 250, 256, 257, 512, 513, 1000, 1001, 1024, 1026, 2048, 2056, 4096, 4100, 4102, 8192, 8193]


def pick(t, form):
    keep = {k: v for k, v in t.items() if k == 'y' or (form.get(k, 0) != 0)}
    if form.get('gate') is not None:
        keep['gate'] = t['gate']
    if isinstance(form.get('scale'), float):
        keep['scale'] = form['scale']
    return keep


@pytest.mark.parametrize('dtype', [BF, HF, F])
@pytest.mark.parametrize('D', WIDTHS)
def test_forward_and_backward(D, dtype):
    for i, form in enumerate(FORMS):
        t, dout, dz = make([1, 5, 67, 700 if D < 3000 else 300, 4, 33][i], D, dtype, [F, dtype][i % 2], seed=i)
        run_and_check(pick(t, form), dout, dz, bool(form['post']), form.get('gate') or None)


@pytest.mark.parametrize('dtype,D', [(BF, 20001), (BF, 8200), (F, 10000)])
def test_wide_rows(dtype, D):
    """Wider than the registers of a CTA: several looks at each row."""
    test_forward_and_backward(D, dtype)


def test_gradients_of_one_result_and_of_single_leaves():
    from b200gdn import residual_rms_norm
    for D, upstream in itertools.product((64, 1001, 2048, 9000), (('out',), ('z',))):
        t, dout, dz = make(9, D, F, F, seed=1)
        run_and_check(t, dout, dz, True, 'silu', upstream=upstream)
        run_and_check(pick(t, FORMS[1]), dout, dz, False, None, upstream=upstream)
    t, dout, _ = make(9, 512, BF, F, seed=2)
    every = {k: v.clone().requires_grad_(True) for k, v in t.items()}
    want = dict(zip(NAMES, torch.autograd.grad(call(every, True, 'sigmoid')[0], [every[k] for k in NAMES], dout)))
    for k in NAMES:
        one = {n: v.clone().requires_grad_(n == k) for n, v in t.items()}
        assert torch.equal(torch.autograd.grad(call(one, True, 'sigmoid')[0], one[k], dout)[0], want[k])
    # the sum alone: its gradient is both terms'
    y, r = (t[k].clone().requires_grad_(True) for k in ('y', 'residual'))
    a, b = torch.autograd.grad(residual_rms_norm(y, None, r)[0], [y, r], dout)
    assert torch.equal(a, b)
    y = t['y'].clone()
    assert torch.equal(torch.autograd.grad(residual_rms_norm(y, None, r)[0], r, dout)[0], b)


def test_gradient_of_differences():
    """In fp32 along a direction, (f(x + h d) - f(x - h d)) / 2h with h = 2^-6: the third derivative leaves about h^2 of the value's own
    size (2.4e-4), rounding 2^-24 / h x sqrt(terms): 2e-3 in all."""
    t, dout, dz = make(9, 515, F, F, seed=4)
    d = {k: 0.3 * torch.randn_like(v) for k, v in t.items()}
    leaves = {k: v.clone().requires_grad_(True) for k, v in t.items()}
    got = torch.autograd.grad(call(leaves, True, 'silu'), [leaves[k] for k in NAMES], [dout, dz])
    parts = [(g.double() * d[k]).sum() for k, g in zip(NAMES, got)]

    def f(h):
        out, z = call({k: v + h * d[k] for k, v in t.items()}, True, 'silu')
        return (out.double() * dout).sum() + (z.double() * dz).sum()
    h = 2.0 ** -6
    scale = sum((g.double() * d[k]).square().sum() for k, g in zip(NAMES, got)).sqrt() + sum(p.abs() for p in parts)
    assert abs((f(h) - f(-h)) / (2 * h) - sum(parts)) < 2e-3 * scale


@pytest.mark.parametrize('dtype', [BF, F])
def test_rows_of_zeros_and_of_large_values(dtype):
    """A row of zeros stays zero (eps holds the norms); squares of values of 1e18 leave the range that their mean is within."""
    for D in (64, 1001, 2048, 8192, 12000):
        t, dout, dz = make(6, D, dtype, F, seed=5)
        t['y'][1] = 0
        t['residual'][1] = 0
        t['y'][2] = 0
        t['y'][3] *= 1e18
        t['residual'][4] *= 1e18
        out, z = call(t, True, 'sigmoid')
        want = O.rms_norms(t['y'], t['weight'], t['residual'], True, t['post_weight'], t['gate'], 'sigmoid', t['scale'], 1e-6)
        close('out', out, want['out'], want['out_size'])
        close('z', z, want['z'], want['z_size'])
        assert (out[1] == 0).all() and (z[1] == 0).all()


def test_rows_that_are_not_finite_stay_alone():
    for D in (64, 513, 2048, 8200):
        t, dout, dz = make(40, D, BF, F, seed=6)
        clean = call(t, True, 'silu')
        t['y'][7, D // 2] = float('nan')
        t['residual'][11, 0] = float('inf')
        t['gate'][30, D - 1] = float('nan')
        leaves = {k: v.clone().requires_grad_(True) for k, v in t.items()}
        out = call(leaves, True, 'silu')
        rows = [r for r in range(40) if r not in (7, 11, 30)]
        assert all(torch.equal(a[rows].detach(), b[rows]) for a, b in zip(out, clean))
        dy, dres, dgate = torch.autograd.grad(out, [leaves[k] for k in ('y', 'residual', 'gate')], [dout, dz])
        assert all(torch.isfinite(g[rows]).all() for g in (dy, dres, dgate))
        assert torch.isnan(out[0][7]).all() and torch.isnan(out[0][30]).all()


def test_strides_streams_graphs_and_traces():
    from b200gdn import ResidualRMSNorm, residual_rms_norm
    t, dout, dz = make(24, 96, BF, F, seed=7)
    want = call(t, True, 'sigmoid')
    apart = {k: torch.stack([v, v], 1)[:, 0] if v.dim() == 2 else torch.stack([v, v], 1)[:, 0] for k, v in t.items()}
    assert all(torch.equal(a, b) for a, b in zip(call(apart, True, 'sigmoid'), want))
    shaped = {k: v.view(2, 3, 4, 96) if v.dim() == 2 else v for k, v in t.items()}
    assert all(torch.equal(a.view(24, 96), b) for a, b in zip(call(shaped, True, 'sigmoid'), want))

    def both(t):
        leaves = {k: v.detach().requires_grad_(True) for k, v in t.items()}
        out = call(leaves, True, 'sigmoid')
        return [o.detach() for o in out] + list(torch.autograd.grad(out, [leaves[k] for k in NAMES], [dout, dz]))
    other, _, _ = make(24, 96, BF, F, seed=8)
    ref = [both(t), both(other)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both(t)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, ref[0]))
    held, graph = {k: v.clone() for k, v in t.items()}, torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both(held)
    for new, r in ((other, ref[1]), (t, ref[0])):
        for k, v in new.items():
            held[k].copy_(v)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, r))
    m = ResidualRMSNorm(96, post_norm=True, scale=0.5, gate_activation='sigmoid').cuda()
    assert set(m.state_dict()) == {'weight', 'post_weight', 'scale'} and not list(ResidualRMSNorm(96, elementwise_affine=False).parameters())
    x = torch.randn(3, 5, 96, device='cuda')
    got = m(x, x, x)
    assert all(torch.equal(a, b) for a, b in zip(got, residual_rms_norm(x, m.weight, x, True, m.post_weight, x, 'sigmoid', m.scale)))
    w, held = m.weight, m.weight.detach()
    traced = torch.jit.trace(lambda a, b: residual_rms_norm(a, held, b)[0], (x, x))
    new = torch.randn(2, 7, 96, device='cuda')
    assert torch.equal(traced(new, new), residual_rms_norm(new, w, new)[0])
    e = torch.zeros(0, 96, device='cuda', requires_grad=True)
    out, z = residual_rms_norm(e, w, e)
    assert out.shape == (0, 96) and (torch.autograd.grad(out, w, out)[0] == 0).all()


def test_many_rows():
    """More rows than CTAs' turns and offsets beyond 2^31 elements."""
    from b200gdn import residual_rms_norm
    rows, D = 300000, 8192
    y = torch.ones(rows, D, dtype=BF, device='cuda')
    t, _, _ = make(64, D, BF, BF, seed=9)
    y[-64:] = t['y']
    out, z = residual_rms_norm(y, t['weight'], post_norm=True)
    want = O.rms_norms(t['y'], t['weight'], None, True, None, None, None, None, 1e-6)
    close('out', out[-64:], want['out'], want['out_size'])
    close('z', z[-64:], want['z'], want['z_size'])


@pytest.mark.parametrize('dtype', [BF, F])
@pytest.mark.parametrize('D', [10, 1002, 2048])
def test_tensors_at_any_element_of_a_buffer(D, dtype):
    """By the C ABI, which copies nothing."""
    from b200gdn import _lib
    lib, rows = _lib.load(), 19
    code = {F: 0, BF: 1}
    for ptype in (F, BF):
        for i, (xo, po) in enumerate([(0, 1), (0, 2), (1, 0), (2, 3), (4, 4), (0, 0)]):
            t, dout, dz = make(rows, D, dtype, ptype, seed=i)

            def at(v):
                off = xo if v.dim() == 2 else po
                buf = torch.zeros(v.numel() + off + 8, dtype=v.dtype, device='cuda')
                buf[off:off + v.numel()] = v.flatten()
                return buf[off:off + v.numel()].view(v.shape)
            x = {k: at(v) for k, v in dict(t, dout=dout, dz=dz).items()}
            rstd = torch.zeros(2, rows, device='cuda')
            x.update(z=at(torch.zeros_like(dout)), out=at(torch.zeros_like(dout)), rstd_y=rstd[0], rstd_z=rstd[1],
                     partials=torch.zeros(lib.b200gdn_rms_norms_partials(rows, D), device='cuda'))
            x.update({'d' + k: at(torch.zeros_like(t[k])) for k in NAMES})
            a = _lib.RmsNormsArgs(struct_bytes=C.sizeof(_lib.RmsNormsArgs), D=D, rows=rows, dtype=2 if dtype == F else 0, param_dtype=code[ptype],
                                  flags=_lib.NORMS_POST | _lib.NORMS_SILU, eps=1e-6, alpha=1.0, **{k: v.data_ptr() for k, v in x.items()})
            stream = torch.cuda.current_stream().cuda_stream
            assert lib.b200gdn_rms_norms_fwd(C.byref(a), stream) == 0 and lib.b200gdn_rms_norms_bwd(C.byref(a), stream) == 0
            want = O.rms_norms(t['y'], t['weight'], t['residual'], True, t['post_weight'], t['gate'], 'silu', t['scale'], 1e-6, dout, dz)
            for k in ('out', 'z') + tuple('d' + k for k in NAMES):
                close(k, x[k], want[k], want[k + '_size'])


def test_refusals():
    from b200gdn import B200GDNError, ResidualRMSNorm, residual_rms_norm
    x = torch.randn(3, 8, device='cuda')
    for bad, match in ((lambda: residual_rms_norm(x.double()), 'not supported'), (lambda: residual_rms_norm(x[:, :0]), 'without elements'),
                       (lambda: residual_rms_norm(x, x[0, :7]), 'vectors'), (lambda: residual_rms_norm(x, scale=x), 'vectors'),
                       (lambda: residual_rms_norm(x, post_norm=True, post_weight=x[:, 0]), 'vectors'), (lambda: residual_rms_norm(x, x[0].long()), 'vectors'),
                       (lambda: residual_rms_norm(x, x[0].cpu()), 'is on cpu'), (lambda: residual_rms_norm(x, residual=x.cpu()), 'is on cpu'),
                       (lambda: residual_rms_norm(x, residual=x.half()), 'shape and the type'), (lambda: residual_rms_norm(x, gate=x[:1]), 'shape and the type'),
                       (lambda: residual_rms_norm(x.cpu()), 'CUDA device only')):
        with pytest.raises(B200GDNError, match=match):
            bad()
    for bad, match in ((lambda: residual_rms_norm(x, gate=x, gate_activation='tanh'), 'Unsupported'), (lambda: ResidualRMSNorm(8, gate_activation='x'), 'Unsupported'),
                       (lambda: residual_rms_norm(x, post_weight=x[0]), 'post_norm'), (lambda: residual_rms_norm(x, gate_activation='silu'), 'without a `gate`')):
        with pytest.raises(ValueError, match=match):
            bad()
    leaf = x.clone().requires_grad_(True)
    dx, = torch.autograd.grad(residual_rms_norm(leaf)[0].square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match='no second derivative'):
        dx.sum().backward()


def test_the_gradient_of_many_rows():
    """Offsets beyond 2^31 elements, backward."""
    from b200gdn import residual_rms_norm
    rows, D, n = 300000, 8192, 64
    t, dout, dz = make(n, D, BF, F, seed=5)

    def behind(v):   # the last rows of a large tensor
        big = torch.ones(rows, D, dtype=BF, device='cuda')
        big[-n:] = v
        return big
    big = {k: behind(t[k]).requires_grad_(True) for k in ('y', 'residual', 'gate')}
    out, z = residual_rms_norm(big['y'], t['weight'], big['residual'], True, t['post_weight'], big['gate'], 'silu')
    del out
    got = dict(zip(big, torch.autograd.grad([z], list(big.values()), [behind(dz)])))
    want = O.rms_norms(t['y'], t['weight'], t['residual'], True, t['post_weight'], t['gate'], 'silu', None, 1e-6, None, dz)
    for k, v in got.items():
        close('d' + k, v[-n:], want['d' + k], want['d' + k + '_size'])
