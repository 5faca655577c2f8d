"""Layer norm with the residual sum on the GPU against the 64-bit restatement.

Tolerances: a result is rounded once to its type (half a unit: 2^-9 bf16, 2^-12 fp16 and 2^-25 fp32 relative would do; twice
that is allowed), and what is computed in 32 bits before may be off by a few units (2^-24) of the magnitudes it is made of: the sums of a
row run over at most some thousands of terms in short chains, for which 32 units are allowed."""
import pytest
import torch

from oracle import head_oracle as H

pytestmark = pytest.mark.gpu
EPS = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 1e-38, torch.float16: 2.0 ** -24, torch.float32: 1e-38}
UNITS = 32 * 2.0 ** -24


def close(name, got, want, size):
    limit = EPS[got.dtype] * want.abs() + UNITS * size + TINY[got.dtype]
    off = (got.double() - want).abs() / limit
    assert torch.isfinite(got).all(), name
    assert off.max() <= 1.0, f'{name}: {off.max().item():.2f} of what is allowed'


def make(rows, D, dtype, ptype, residual, bias, weight=True, seed=0):
    g = torch.Generator(device='cuda').manual_seed(seed)

    def rn(*s):
        return torch.randn(*s, device='cuda', generator=g)
    x = (rn(rows, D) + 0.5).to(dtype)
    res = (3 * rn(rows, D)).to(dtype) if residual else None
    w = (1 + 0.3 * rn(D)).to(ptype) if weight else None
    b = rn(D).to(ptype) if bias else None
    return x, w, b, res, rn(rows, D).to(dtype), rn(rows, D).to(dtype)


WIDTHS = [1, 2, 7, 8, 33, 64, 100, 128, 250, 256, 511, 512, 768, 1000, 1001, 1024, 1026, 2048, 2056, 4096, 4100, 5000, 8192, 8200, 16384, 20001]


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize('D', WIDTHS)
def test_forward_and_backward(D, dtype):
    from b200gdn import layer_norm
    for i, (rows, residual, bias) in enumerate([(1, False, True), (5, True, False), (67, True, True), (700 if D < 3000 else 300, False, False)]):
        ptype = [torch.float32, dtype][i % 2]
        x, w, b, res, dy, dz = make(rows, D, dtype, ptype, residual, bias, weight=i != 3, seed=i)
        leaves = [t.requires_grad_(True) for t in (x, w, b, res) if t is not None]
        out = layer_norm(x, w, b, residual=res, prenorm=residual)
        out = out if residual else (out,)
        grads = torch.autograd.grad(out, leaves, [dy, dz][:len(out)])
        want = H.layer_norm(x.detach(), *(None if t is None else t.detach() for t in (w, b, res)), 1e-5, dy, dz if residual else None)
        close('y', out[0].detach(), want['y'], want['y_size'])
        got = dict(zip([n for n, t in zip(('x', 'w', 'b', 'res'), (x, w, b, res)) if t is not None], grads))
        close('dx', got['x'], want['dx'], want['dx_size'])
        if residual:
            assert torch.equal(out[1].detach(), want['z']) and torch.equal(got['res'], got['x'])
        if w is not None:
            close('dweight', got['w'], want['dweight'], want['dweight_size'])
        if bias:
            close('dbias', got['b'], want['dbias'], want['dbias_size'])
        with torch.no_grad():   # the forward pass alone gives the same
            again = layer_norm(x, w, b, residual=res, prenorm=residual)
            assert torch.equal(again[0] if residual else again, out[0])
            if residual:
                assert torch.equal(layer_norm(x, w, b, residual=res), out[0])


@pytest.mark.parametrize('dtype,D', [(torch.bfloat16, 40000), (torch.bfloat16, 10002), (torch.float32, 20000), (torch.float32, 9001)])
def test_wide_rows(D, dtype):
    """Wider than the registers of a CTA, forward or backward."""
    test_forward_and_backward(D, dtype)


def test_gradient_of_differences():
    """In fp32, along a direction: (f(x + h d) - f(x - h d)) / 2h.  With h = 2^-6 the third derivative leaves about h^2 / 6 of the
    value's own size (4e-5 of it; y is smooth on the scale of a row's spread), rounding 2^-24 / h x sqrt(terms): 1e-3 in all."""
    from b200gdn import layer_norm
    x, w, b, res, dy, _ = make(9, 515, torch.float32, torch.float32, True, True, seed=4)
    d = [torch.randn_like(t) for t in (x, w, b, res)]
    leaves = [t.requires_grad_(True) for t in (x, w, b, res)]
    grads = torch.autograd.grad(layer_norm(x, w, b, residual=res), leaves, dy)
    h = 2.0 ** -6
    for i in range(4):
        def f(sign):
            args = [t.detach() + (sign * h * d[i] if j == i else 0) for j, t in enumerate(leaves)]
            return (layer_norm(args[0], args[1], args[2], residual=args[3]).double() * dy).sum()
        want, got = ((f(1) - f(-1)) / (2 * h)).item(), (grads[i].double() * d[i]).sum().item()
        assert abs(got - want) < 1e-3 * (grads[i].double() * d[i]).norm().item() * 3 + 1e-3


def test_which_gradients_are_asked_for():
    from b200gdn import layer_norm
    x, w, b, res, dy, dz = make(40, 256, torch.bfloat16, torch.float32, True, True)
    want = H.layer_norm(x, w, b, res, 1e-5, dy, dz)
    for need in range(1, 16):
        leaves = [t.detach().requires_grad_(bool(need >> i & 1)) for i, t in enumerate((x, w, b, res))]
        y, z = layer_norm(leaves[0], leaves[1], leaves[2], residual=leaves[3], prenorm=True)
        if z.requires_grad:
            torch.autograd.backward([y, z], [dy, dz])
        else:
            y.backward(dy)
        for t, n in zip(leaves, ('dx', 'dweight', 'dbias', 'dx')):
            assert (t.grad is None) == (not t.requires_grad)
            if t.grad is not None and z.requires_grad:
                close(n, t.grad, want[n], want[n + '_size'])
    # only one of the two results is used
    leaf = x.detach().requires_grad_(True)
    y, z = layer_norm(leaf, w, b, residual=res, prenorm=True)
    assert torch.equal(torch.autograd.grad(z, leaf, dz, retain_graph=True)[0], dz)
    only = H.layer_norm(x, w, b, res, 1e-5, dy)
    close('dx', torch.autograd.grad(y, leaf, dy)[0], only['dx'], only['dx_size'])
    # the one tensor as x and as residual
    both = x.detach().float().requires_grad_(True)
    got, = torch.autograd.grad(layer_norm(both, w, b, residual=both), both, dy.float())
    twice = H.layer_norm(both.detach(), w, b, both.detach(), 1e-5, dy.float())
    close('dx', got, 2 * twice['dx'], 2 * twice['dx_size'])


def test_rows_of_any_kind():
    """Constant rows, huge and tiny ones, infinities and NaN, strided and unaligned tensors, leading dimensions, no rows."""
    from b200gdn import layer_norm
    dev = 'cuda'
    x = torch.zeros(6, 640, device=dev)
    x[1] = 3.0
    x[2] = 1e18 * torch.randn(640, device=dev)
    x[3] = 1e-18 * torch.randn(640, device=dev)
    x[4] = torch.randn(640, device=dev)
    x[4, 17] = float('inf')
    x[5] = torch.randn(640, device=dev)
    x[5, 3] = float('nan')
    y = layer_norm(x)
    want = H.layer_norm(x[:4], None, None, None, 1e-5)
    assert (y[:2] == 0).all()
    close('y', y[2:4], want['y'][2:4], want['y_size'][2:4])
    assert y[4:].isnan().all()
    base = torch.randn(5, 3, 1003, device=dev).to(torch.bfloat16)
    for v in (base[:, 1:, 2:900], base.transpose(0, 1), base.flatten()[5:5 + 998 * 3].view(3, 998)):
        want = H.layer_norm(v.reshape(-1, v.shape[-1]), None, None, None, 1e-5)
        got = layer_norm(v)
        assert got.shape == v.shape
        close('y', got.reshape(-1, v.shape[-1]), want['y'], want['y_size'])
    none = torch.zeros(0, 7, device=dev, requires_grad=True)
    w = torch.ones(7, device=dev, requires_grad=True)
    y = layer_norm(none, w)
    y.sum().backward()
    assert y.shape == (0, 7) and none.grad.shape == (0, 7) and (w.grad == 0).all()


def test_results_do_not_depend_on_the_run():
    from b200gdn import layer_norm
    x, w, b, res, dy, dz = make(3001, 1024, torch.bfloat16, torch.float32, True, True)
    runs = []
    for _ in range(3):
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b, res)]
        out = layer_norm(leaves[0], leaves[1], leaves[2], residual=leaves[3], prenorm=True)
        runs.append([*out, *torch.autograd.grad(out, leaves, [dy, dz])])
    for r in runs[1:]:
        assert all(torch.equal(p, q) for p, q in zip(r, runs[0]))


def test_module_stream_graph_and_trace():
    from b200gdn import LayerNorm
    torch.manual_seed(0)
    m = LayerNorm(512, bias=True, device='cuda')
    x, res = torch.randn(33, 512, device='cuda'), torch.randn(33, 512, device='cuda')
    with torch.no_grad():
        m.weight.normal_()
        m.bias.normal_()
        want = m(x, res, True)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = m(x, res, True)
        side.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = m(x, res, True)
        x.normal_()
        graph.replay()
        assert all(torch.equal(p, q) for p, q in zip(got, m(x, res, True)))
        assert set(m.state_dict()) == {'weight', 'bias'} and LayerNorm(4, elementwise_affine=False).weight is None
        y, z = m(x, None, True)
        assert z is x
    traced = torch.jit.trace(m, (x,))
    other = torch.randn(5, 512, device='cuda')
    assert torch.equal(traced(other), m(other))


def test_refusals():
    from b200gdn import B200GDNError, layer_norm
    x = torch.randn(3, 8, device='cuda')
    with pytest.raises(B200GDNError, match='CUDA device only'):
        layer_norm(x.cpu())
    with pytest.raises(B200GDNError, match='not supported'):
        layer_norm(x.double())
    with pytest.raises(B200GDNError, match='without elements'):
        layer_norm(x[:, :0])
    with pytest.raises(B200GDNError, match='weight and bias'):
        layer_norm(x, x[0, :7])
    with pytest.raises(B200GDNError, match='weight and bias'):
        layer_norm(x, x[0], x[:, 0])
    with pytest.raises(B200GDNError, match='is on cpu'):
        layer_norm(x, x[0].cpu())
    with pytest.raises(B200GDNError, match='shape and the type'):
        layer_norm(x, residual=x.half())
    with pytest.raises(B200GDNError, match='shape and the type'):
        layer_norm(x, residual=x.view(4, 6))
    leaf = x.clone().requires_grad_(True)
    dx, = torch.autograd.grad(layer_norm(leaf).square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match='no second derivative'):
        dx.sum().backward()


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('D', [10, 1002, 2048])
def test_tensors_at_any_element_of_a_buffer(D, dtype):
    """By the C ABI, which copies nothing: rows and fp32 or 16-bit parameters that begin one, two or four elements into their buffers."""
    import ctypes as C
    from b200gdn import _lib
    lib, rows = _lib.load(), 19
    code = {torch.float32: 0, torch.bfloat16: 1}
    for ptype in (torch.float32, torch.bfloat16):
        for i, (xo, wo, bo) in enumerate([(0, 1, 0), (0, 0, 1), (0, 2, 2), (2, 1, 3), (1, 0, 0), (4, 4, 4), (0, 3, 5), (0, 0, 0)]):
            x, w, b, _, dy, _ = make(rows, D, dtype, ptype, False, True, seed=i)

            def at(t, off):
                buf = torch.zeros(t.numel() + off + 8, dtype=t.dtype, device='cuda')
                buf[off:off + t.numel()] = t.flatten()
                return buf[off:off + t.numel()].view(t.shape)
            x, w, b, dy = at(x, xo), at(w, wo), at(b, bo), at(dy, xo)
            y, dx = at(torch.zeros_like(x), xo), at(torch.zeros_like(x), xo)
            mean, rstd = torch.zeros(rows, device='cuda'), torch.zeros(rows, device='cuda')
            dw, db = at(torch.zeros_like(w), wo), at(torch.zeros_like(b), bo)
            partials = torch.zeros(lib.b200gdn_layer_norm_ctas(rows) * 2 * D, device='cuda')
            shape = dict(struct_bytes=C.sizeof(_lib.LayerNormArgs), D=D, rows=rows, dtype=2 if dtype == torch.float32 else 0, param_dtype=code[ptype], eps=1e-5)
            p = {k: v.data_ptr() for k, v in dict(x=x, w=w, b=b, y=y, mean=mean, rstd=rstd, dy=dy, dx=dx, dw=dw, db=db, partials=partials).items()}
            stream = torch.cuda.current_stream().cuda_stream
            assert lib.b200gdn_layer_norm_fwd(C.byref(_lib.LayerNormArgs(x=p['x'], weight=p['w'], bias=p['b'], y=p['y'], mean=p['mean'], rstd=p['rstd'], **shape)), stream) == 0
            assert lib.b200gdn_layer_norm_bwd(C.byref(_lib.LayerNormArgs(z=p['x'], weight=p['w'], mean=p['mean'], rstd=p['rstd'], dy=p['dy'], dx=p['dx'],
                                                                         dweight=p['dw'], dbias=p['db'], partials=p['partials'], **shape)), stream) == 0
            want = H.layer_norm(x, w, b, None, 1e-5, dy)
            for name, got in (('y', y), ('dx', dx), ('dweight', dw), ('dbias', db)):
                close(name, got, want[name], want[name + '_size'])


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize('D', [1, 2, 8, 64, 256, 512, 1024, 2048, 4096, 8192, 16384, 32768, 65536])
def test_constant_rows(D, dtype):
    """Rows of one value v of at most 8 bits: sums of a power of two of them and their mean are exact, and z - mean is zero.  So y is
    the bias, the weight's gradient zero and dx = rstd (h - mean(h)), whatever eps makes of rstd."""
    from b200gdn import layer_norm
    v = torch.tensor([0.1, 100.0, 1000.0, -7.3, 0.0, 3.0, 1e-3]).bfloat16().float().cuda()
    x = v[:, None].expand(len(v), D).to(dtype).contiguous().requires_grad_(True)
    x_half = (x.detach().float() / 2).to(dtype)   # (exact) twice that, as a residual sum
    w = (1 + 0.3 * torch.randn(D, device='cuda', generator=torch.Generator('cuda').manual_seed(0))).requires_grad_(True)
    b = torch.randn(D, device='cuda', generator=torch.Generator('cuda').manual_seed(1)).requires_grad_(True)
    dy = torch.randn(len(v), D, device='cuda', generator=torch.Generator('cuda').manual_seed(2)).to(dtype)
    h = dy.double() * w.detach().double()
    for eps in (1e-5, 1e-12):
        r = eps ** -0.5
        for y in (layer_norm(x, w, b, eps=eps), layer_norm(x_half.requires_grad_(True), w, b, residual=x_half, eps=eps)):
            assert torch.equal(y.detach(), b.detach().to(dtype).expand_as(y))
        dx, dw = torch.autograd.grad(layer_norm(x, w, b, eps=eps), [x, w], dy)
        assert (dw == 0).all()
        if dtype is not torch.float16 or eps == 1e-5:   # (1e6 leaves what fp16 holds)
            close('dx', dx, r * (h - h.mean(-1, keepdim=True)), r * (h.abs() + h.abs().mean(-1, keepdim=True)))
