"""Projections on the GPU against the 64-bit restatement.

Tolerances: a result is rounded once to its type (half a step of the type, allowed twice: bf16 2^-8, fp16 2^-11 relative), and what is
computed before may be off by what oracle/block_oracle.py derives."""
import pytest
import torch

from oracle import block_oracle as O

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
EPS = {BF: 2.0 ** -8, HF: 2.0 ** -11}
TINY = {BF: 1e-37, HF: 2.0 ** -24}


def close(name, got, want, off):
    limit = EPS[got.dtype] * want.abs() + off + TINY[got.dtype]
    assert torch.isfinite(got).all(), name
    if got.numel():
        far = ((got.double() - want).abs() / limit).max().item()
        assert far <= 1.0, f'{name}: {far:.2f} of what is allowed'


def make(M, K, N, dtype, bias=True, residual=True, seed=0):
    gen = torch.Generator(device='cuda').manual_seed(seed)

    def rn(*s, scale=1.0):
        return (scale * torch.randn(*s, device='cuda', generator=gen)).to(dtype)
    return rn(M, K), rn(N, K, scale=K ** -0.5), rn(N) if bias else None, rn(M, N) if residual else None, rn(M, N)


NAMES = ('x', 'weight', 'bias', 'residual')


def run_and_check(M, K, N, dtype, act, bias, residual, seed=0):
    from b200gdn import fused_linear
    *tensors, dy = make(M, K, N, dtype, bias, residual, seed)
    leaves = [None if t is None else t.clone().requires_grad_(True) for t in tensors]
    y = fused_linear(*leaves, activation=act)
    want = O.linear(*tensors, act, dy)
    close('y', y.detach(), want['y'], want['y_off'])
    got = torch.autograd.grad(y, [t for t in leaves if t is not None], dy)
    for name, g in zip([n for n, t in zip(NAMES, leaves) if t is not None], got):
        if name == 'residual':
            assert torch.equal(g, dy)
        else:
            close('d' + name, g, want['d' + name], want['d' + name + '_off'])
    with torch.no_grad():
        assert torch.equal(fused_linear(*tensors, activation=act), y)


FORMS = [('silu', True, False), (None, False, True), ('gelu', True, True), ('sigmoid', False, False), (None, True, False)]


@pytest.mark.parametrize('K,N', [(64, 64), (8, 16), (1, 1), (7, 9), (136, 104), (1003, 130), (96, 2050), (2048, 512), (512, 2048)])
@pytest.mark.parametrize('M', [1, 2, 3, 8, 9, 33, 64, 65, 129, 200, 256, 257, 300, 1021])
def test_forward_and_backward(M, K, N):
    for i, dtype in enumerate((BF, HF)):
        act, bias, residual = FORMS[(M + N + i * 2) % 5]
        run_and_check(M, K, N, dtype, act, bias, residual, seed=i)


@pytest.mark.parametrize('act', [None, 'silu', 'sigmoid', 'gelu'])
@pytest.mark.parametrize('M', [4, 100, 600])
def test_every_activation(M, act):
    for dtype, K, N in ((BF, 256, 384), (HF, 255, 129)):
        run_and_check(M, K, N, dtype, act, True, True)


@pytest.mark.parametrize('M,K,N', [(20000, 64, 48), (700, 6000, 300), (300, 40, 9000), (5000, 520, 1000), (12, 20000, 30), (250, 8192, 2048)])
def test_long_sides(M, K, N):
    """Many tiles for a CTA pair, a contraction in parts, one that fills no step."""
    run_and_check(M, K, N, BF, 'silu', True, False)
    run_and_check(M, K, N, BF, None, False, True)


def test_gradient_of_differences():
    """fp16 along a direction in the loss of a smooth activation: (f(x + h d) - f(x - h d)) / 2h with h d representable.  Rounding of y by half a
    step (2^-11) of each of M N terms, added in quadrature (factor sqrt(2) / 2h), and h^2 / 6 of the third derivative's size."""
    from b200gdn import fused_linear
    M, K, N = 40, 72, 88
    x, w, b, r, dy = make(M, K, N, HF)
    h = 2.0 ** -4
    d = torch.randint(-1, 2, (M, K), device='cuda').to(HF)
    x = (x * 16).round() / 16   # (so that x + h d is exact)
    leaf = x.clone().requires_grad_(True)
    y = fused_linear(leaf, w, b, r, 'silu')
    g, = torch.autograd.grad(y, leaf, dy)
    along = (g.double() * d).sum()

    def f(e):
        return (fused_linear(x + e * d, w, b, r, 'silu').double() * dy.double()).sum()
    step = (d.double() @ w.double().t())
    rounding = (y.detach().double().abs() * dy.double().abs() * 2.0 ** -11).square().sum().sqrt() / h
    third = (h * h / 6) * (step.abs() ** 3 * dy.double().abs()).sum() * 0.5
    own = (g.double().abs() * 2.0 ** -10 * d.double().abs()).sum()
    assert abs((f(h) - f(-h)) / (2 * h) - along) < 4 * rounding + third + own


def test_values_that_are_not_finite_stay_with_their_token():
    from b200gdn import fused_linear
    for M in (5, 100, 400):
        x, w, b, r, dy = make(M, 200, 72, BF)
        clean = fused_linear(x, w, b, r)
        x[3, 7] = float('nan')
        bad = fused_linear(x, w, b, r)
        keep = [i for i in range(M) if i != 3]
        assert torch.equal(bad[keep], clean[keep]) and torch.isnan(bad[3]).all()


def test_shapes_strides_streams_graphs_traces_and_module():
    from b200gdn import FusedLinear, fused_linear
    x, w, b, r, dy = make(24, 96, 80, BF)
    want = fused_linear(x, w, b, r, 'silu')
    assert torch.equal(fused_linear(x.view(2, 3, 4, 96), w, b, r.view(2, 3, 4, 80), 'silu').view(24, 80), want)
    assert torch.equal(fused_linear(x.t().contiguous().t(), w.t().contiguous().t(), b, r.t().contiguous().t(), 'silu'), want)
    assert torch.equal(fused_linear(x[3], w, b, r[3]), fused_linear(x[3:4], w, b, r[3:4])[0])
    for off in (1, 3, 8):   # at any element of a buffer
        def at(t):
            buf = torch.zeros(t.numel() + off, dtype=t.dtype, device='cuda')
            buf[off:] = t.flatten()
            return buf[off:].view(t.shape)
        assert torch.equal(fused_linear(at(x), at(w), at(b), at(r), 'silu'), want)
    for M in (4, 70, 700):
        data = [make(M, 136, 104, BF, seed=s) for s in (1, 2)]

        def both(x, w, b, r, dy):
            leaves = [t.detach().requires_grad_(True) for t in (x, w, b, r)]
            y = fused_linear(*leaves, activation='gelu')
            return [y.detach(), *torch.autograd.grad(y, leaves, dy)]
        ref = [both(*d) for d in data]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = both(*data[0])
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(p, q) for p, q in zip(got, ref[0]))
        held, graph = [t.clone() for t in data[0]], torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = both(*held)
        for d, want_ in ((data[1], ref[1]), (data[0], ref[0])):
            for t, n in zip(held, d):
                t.copy_(n)
            graph.replay()
            assert all(torch.equal(p, q) for p, q in zip(got, want_))
    m = FusedLinear(96, 80, activation='silu').cuda().to(BF)
    assert set(m.state_dict()) == {'weight', 'bias'} and FusedLinear(8, 8, bias=False).bias is None
    assert torch.equal(m(x, r), fused_linear(x, m.weight, m.bias, r, 'silu'))
    traced = torch.jit.trace(lambda a, c: fused_linear(a, w, b, c, 'silu'), (x, r))
    y, _, _, s, _ = make(300, 96, 80, BF, seed=4)
    assert torch.equal(traced(y, s), fused_linear(y, w, b, s, 'silu'))
    e = torch.zeros(0, 96, device='cuda', dtype=BF, requires_grad=True)
    out = m(e)
    assert out.shape == (0, 80)
    assert all((g == 0).all() for g in torch.autograd.grad(out, [m.weight, m.bias], out))


def test_gradients_of_single_leaves():
    from b200gdn import fused_linear
    for M in (6, 300):
        *tensors, dy = make(M, 64, 40, BF)
        every = [t.clone().requires_grad_(True) for t in tensors]
        want = torch.autograd.grad(fused_linear(*every, activation='silu'), every, dy)
        for i in range(4):
            one = [t.clone().requires_grad_(k == i) for k, t in enumerate(tensors)]
            assert torch.equal(torch.autograd.grad(fused_linear(*one, activation='silu'), one[i], dy)[0], want[i])


def test_refusals():
    from b200gdn import B200GDNError, FusedLinear, fused_linear
    x, w, b, r, _ = make(6, 16, 24, BF)
    for bad, match in ((lambda: fused_linear(x.float(), w.float()), 'not supported'), (lambda: fused_linear(x, w.half()), 'type of x'),
                       (lambda: fused_linear(x, w, b.float()), 'type of x'), (lambda: fused_linear(x, w[:, :8]), 'weight is'), (lambda: fused_linear(x, w[0]), 'weight is'),
                       (lambda: fused_linear(x, w[:0]), 'weight is'), (lambda: fused_linear(x[:, :0], w[:, :0]), 'without features'),
                       (lambda: fused_linear(x, w, b[:3]), 'bias is'), (lambda: fused_linear(x, w, b, r[:1]), 'residual has'), (lambda: fused_linear(x, w, b, r[0]), 'residual has'),
                       (lambda: fused_linear(x, w.cpu()), 'is on cpu'), (lambda: fused_linear(x.cpu(), w), 'CUDA device only')):
        with pytest.raises(B200GDNError, match=match):
            bad()
    for bad in (lambda: fused_linear(x, w, activation='relu'), lambda: FusedLinear(4, 4, activation='tanh')):
        with pytest.raises(ValueError, match='Unsupported'):
            bad()
    leaf = x.clone().requires_grad_(True)
    dx, = torch.autograd.grad(fused_linear(leaf, w).float().square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match='no second derivative'):
        dx.sum().backward()


def test_calls_of_few_tokens_in_a_row():
    """Each call reads what the one ahead has just written, and begins before it ends: in a captured graph, on changing data, against calls
    between which the device is waited for."""
    from b200gdn import fused_linear
    for M, D in ((1, 1024), (4, 2048), (16, 520), (9, 96)):
        gen = torch.Generator(device='cuda').manual_seed(M)
        layers = [(torch.randn(D, D, device='cuda', generator=gen) * D ** -0.5).to(BF) for _ in range(6)]
        data = [torch.randn(M, D, device='cuda', generator=gen).to(BF) for _ in range(8)]

        def chain(x, wait):
            out = []
            for w in layers:
                x = fused_linear(x, w, None, x, 'silu')
                out.append(x)
                if wait:
                    torch.cuda.synchronize()
            return out
        want = [chain(x, True) for x in data]
        held, graph = data[0].clone(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = chain(held, False)
        for _ in range(3):
            for x, w in zip(data, want):
                held.copy_(x)
                graph.replay()
                assert all(torch.equal(p, q) for p, q in zip(got, w))
                assert all(torch.equal(p, q) for p, q in zip(chain(x, False), w))


@pytest.mark.parametrize('act', ['silu', 'gelu', 'sigmoid'])
@pytest.mark.parametrize('M', [7, 100, 600])
def test_gradients_where_the_activations_input_leaves_the_types_range(M, act):
    """fp16: feature 0 has z = -80000, feature 1 z = 70000, beyond 65504, where the activation is applied all the same: their slopes are 0 and 1 (of the sigmoid 0 and
    0).  Feature 1's y comes back into range by the residual."""
    from b200gdn import fused_linear
    for K, N in ((64, 64), (72, 50), (33, 35)):   # dz by eight, two and one element a thread
        x, w, b, r, dy = make(M, K, N, HF, seed=N)
        x[:, 0] = 250
        w[:, 0] = 0
        w[:2] = 0
        w[0, 0], w[1, 0] = -320, 280
        b[:2], r[:, 1] = 0, -40000 if act != 'sigmoid' else 0
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
        y = fused_linear(*leaves, activation=act)
        want = O.linear(x, w[1:], b[1:], r[:, 1:], act, dy[:, 1:])   # feature 0 adds nothing to any gradient
        close('y', y.detach()[:, 1:], want['y'], want['y_off'])
        assert torch.equal(y.detach()[:, 0], r[:, 0])
        dx, dw, db, _ = torch.autograd.grad(y, leaves, dy)
        close('dx', dx, want['dx'], want['dx_off'])
        assert (dw[0] == 0).all() and db[0] == 0
        close('dweight', dw[2:], want['dweight'][1:], want['dweight_off'][1:])
        close('dbias', db[2:], want['dbias'][1:], want['dbias_off'][1:])
        # (the oracle lets a slope be off by z's rounding, which here it is not)
        up = dy[:, 1].double() * (act != 'sigmoid')
        units = (M / 16 + 32) * 2 * O.U
        close('dweight', dw[1], up @ x.double(), units * (up.abs() @ x.double().abs()))
        close('dbias', db[1], up.sum(), units * up.abs().sum())


@pytest.mark.parametrize('M', [9, 250, 1000])
@pytest.mark.parametrize('dtype', [BF, HF])
def test_gelu_where_little_is_left_of_it(dtype, M):
    """Far below zero, z exact (the weight is the identity).  A result is off by half a step of its type (denormal ones by half of the smallest, 2^-25 in
    fp16) and by what fp32 leaves of erfc: 16 units for the functions and v^2 for the argument's rounding, by their size."""
    from b200gdn import fused_linear
    K = 40
    x = -torch.linspace(0.0, 12.0 if dtype == BF else 5.6, M * K, device='cuda').to(dtype).view(M, K)
    eye = torch.eye(K, device='cuda', dtype=dtype)
    leaf = x.clone().requires_grad_(True)
    y = fused_linear(leaf, eye, activation='gelu')
    dx, = torch.autograd.grad(y, leaf, torch.ones_like(y))
    v = x.double()
    cdf, pdf = 0.5 * torch.special.erfc(-v * 0.5 ** 0.5), torch.exp(-0.5 * v * v) / (2 * torch.pi) ** 0.5
    for name, got, want, size in (('y', y.detach(), v * cdf, v.abs() * cdf), ('dx', dx, cdf + v * pdf, cdf + v.abs() * pdf)):
        limit = EPS[dtype] * want.abs() + (v * v + 16) * 2 * O.U * size + (2.0 ** -25 if dtype == HF else 1e-38)
        far = ((got.double() - want).abs() / limit).max().item()
        assert far <= 1.0, f'{name}: {far:.2f} of what is allowed'


def test_results_of_many_rows():
    """Offsets beyond 2^31 elements, forward and backward: the last rows' results are those of a short call; where the others' upstream gradient is zero, so are
    the sums over all rows."""
    from b200gdn import fused_linear
    M, K, N, n = 300000, 72, 8192, 300
    x, w, b, r, dy = make(n, K, N, BF, seed=6)
    want = O.linear(x, w, b, r, 'silu', dy)

    def behind(v):
        big = torch.zeros(M, v.shape[1], dtype=BF, device='cuda')
        big[-n:] = v
        return big
    leaves = [behind(x).requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True), behind(r)]
    y = fused_linear(*leaves, activation='silu')
    close('y', y.detach()[-n:], want['y'], want['y_off'])
    got = torch.autograd.grad(y, leaves[:3], behind(dy))
    del y
    for name, g in zip(NAMES, got):
        close('d' + name, g[-n:] if name == 'x' else g, want['d' + name], want['d' + name + '_off'])
    assert (got[0][:-n] == 0).all()
    del got, leaves
    x, w, b, r, dy = make(n, N, K, BF, seed=7)   # x and dx of so many elements
    want = O.linear(x, w, b, r, None, dy)
    leaves = [behind(x).requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True)]
    y = fused_linear(*leaves, behind(r))
    close('y', y.detach()[-n:], want['y'], want['y_off'])
    for name, g in zip(NAMES, torch.autograd.grad(y, leaves, behind(dy))):
        close('d' + name, g[-n:] if name == 'x' else g, want['d' + name], want['d' + name + '_off'])
