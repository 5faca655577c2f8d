"""The gated recurrence on the GPU against the 64-bit restatement, token by token.

Tolerances: a result is rounded once to its type (half a step of the type, allowed twice: bf16 2^-8, fp16 2^-11, fp32 2^-24 relative), and
what is computed in 32 bits before may be off by what oracle/block_oracle.py adds up along the sequence."""
import pytest
import torch

from oracle import block_oracle as O

pytestmark = pytest.mark.gpu
EPS = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 1e-37, torch.float16: 2.0 ** -24, torch.float32: 1e-37}
BF, HF, F = torch.bfloat16, torch.float16, torch.float32


def close(name, got, want, off):
    limit = EPS[got.dtype] * want.abs() + off + TINY[got.dtype]
    assert torch.isfinite(got).all(), name
    if got.numel():
        far = ((got.double() - want).abs() / limit).max().item()
        assert far <= 1.0, f'{name}: {far:.2f} of what is allowed'


def make(B, T, D, n_seq, dtype, gtype, h0, seed=0, fast=False):
    gen = torch.Generator(device='cuda').manual_seed(seed)

    def rn(*s):
        return torch.randn(*s, device='cuda', generator=gen)
    x = rn(B, T, D).to(dtype)
    slow = torch.exp(-6 * torch.rand(D, device='cuda', generator=gen))
    g = (-torch.nn.functional.softplus(rn(B, T, D)) * (3.0 if fast else slow)).to(gtype)
    return x, g, (2 * rn(n_seq, D)) if h0 else None, rn(B, T, D).to(dtype), rn(n_seq, D)


def run_and_check(x, g, h0, dh, dht, bounds, cu=None, state=True, grads=('h', 'ht')):
    from b200gdn import gated_recurrence
    kw = dict(cu_seqlens=cu)
    leaves = [t.detach().clone().requires_grad_(True) if t is not None else None for t in (x, g, h0)]
    h, ht = gated_recurrence(leaves[0], leaves[1], initial_state=leaves[2], output_final_state=state, **kw)
    D = x.shape[-1]

    def flat(t):
        return t.reshape(-1, D)
    up_h, up_t = 'h' in grads, state and 'ht' in grads
    want = O.recurrence(flat(x), flat(g), h0, bounds, flat(dh) if up_h else None, dht if up_t else None)
    close('h', flat(h.detach()), want['h'], want['h_off'])
    if state:
        assert ht.dtype == F
        close('ht', ht.detach(), want['ht'], want['ht_off'])
    else:
        assert ht is None
    ins = [t for t in leaves if t is not None]
    got = torch.autograd.grad([h] * up_h + [ht] * up_t, ins, [dh] * up_h + [dht] * up_t)
    for name, t in zip(('dx', 'dg', 'dh0'), got):
        assert t.dtype == (x.dtype if name == 'dx' else g.dtype if name == 'dg' else F)
        close(name, flat(t), want[name], want[name + '_off'])
    with torch.no_grad():   # without gradients the same
        again = gated_recurrence(x, g, initial_state=h0, output_final_state=state, **kw)
    assert torch.equal(again[0], h) and (not state or torch.equal(again[1], ht))
    return h.detach(), ht, got


SHAPES = [(1, 1, 64), (3, 1, 5), (2, 2, 1), (2, 7, 33), (5, 8, 64), (3, 9, 130), (2, 64, 66), (1, 65, 2), (2, 63, 31), (1, 127, 64), (2, 128, 70),
          (2, 129, 96), (3, 257, 130), (1, 1025, 24), (1, 2500, 7), (1, 1500, 64), (2, 700, 200)]


@pytest.mark.parametrize('B,T,D', SHAPES)
@pytest.mark.parametrize('dtype,gtype', [(BF, BF), (BF, F), (HF, HF), (HF, F), (F, F)])
def test_dense(B, T, D, dtype, gtype):
    for h0, fast, seed in ((True, False, 0), (False, True, 1)):
        args = make(B, T, D, B, dtype, gtype, h0, seed, fast)
        run_and_check(*args, O.dense_bounds(B, T), state=h0)


@pytest.mark.parametrize('cu,rows', [([0, 5], 5), ([0, 1, 2, 3], 3), ([0, 0, 1, 9, 9, 300, 1000], 1000), ([0, 64, 128, 129], 129), ([3, 3, 70, 200], 260),
                                     ([0, 16, 600, 616], 616), ([0, 0, 0], 4), ([0, 30, 61, 90, 3000], 3000)])
@pytest.mark.parametrize('D,dtype', [(64, BF), (37, BF), (130, F)])
def test_packed(cu, rows, D, dtype):
    for h0 in (True, False):
        x, g, s, dh, dht = make(1, rows, D, len(cu) - 1, dtype, dtype, h0, seed=len(cu))
        cu_t = torch.tensor(cu, dtype=torch.int32, device='cuda')
        h, _, got = run_and_check(x, g, s, dh, dht, O.packed_bounds(cu), cu=cu_t)
        for t in (h, got[0], got[1]):   # rows that no sequence covers
            assert (t[0, :cu[0]] == 0).all() and (t[0, cu[-1]:] == 0).all()


@pytest.mark.parametrize('D,dtype,gtype', [(1280, BF, BF), (1290, BF, F), (1283, F, F), (1280, HF, F)])
def test_one_sequence_much_longer_than_the_others(D, dtype, gtype):
    """More pieces of work than SMs, and yet the longest sequence is shared by CTAs."""
    cu = [0, 5, 10, 20, 60, 64, 2000, 2010, 2100]
    args = make(1, 2100, D, 8, dtype, gtype, True, seed=20)
    run_and_check(*args, O.packed_bounds(cu), cu=torch.tensor(cu, dtype=torch.int32, device='cuda'))


def test_gradients_of_one_result_only():
    for grads in (('h',), ('ht',)):
        for B, T, D in ((2, 1, 8), (2, 70, 34), (1, 1400, 64)):
            run_and_check(*make(B, T, D, B, F, F, True, seed=3), O.dense_bounds(B, T), grads=grads)


@pytest.mark.parametrize('dtype,gtype', [(BF, BF), (F, F), (HF, F)])
def test_slices_are_read_where_they_lie(dtype, gtype):
    """x and g as halves of one projection, and beginning at any element of a buffer."""
    from b200gdn import gated_recurrence
    for B, T, D, lead in ((2, 130, 64, 0), (2, 33, 50, 1), (3, 1, 64, 2), (1, 1100, 10, 3)):
        x, g, h0, dh, _ = make(B, T, D, B, dtype, gtype, True, seed=5)
        if dtype == gtype:
            wide = torch.empty(B, T, 2 * D + lead, dtype=dtype, device='cuda')
            sx, sg = wide[..., lead:lead + D], wide[..., lead + D:]
        else:
            sx = torch.empty(B, T, D + lead, dtype=dtype, device='cuda')[..., lead:]
            sg = torch.empty(B, T, D + 2 * lead + 1, dtype=gtype, device='cuda')[..., lead:lead + D]
        sx.copy_(x)
        sg.copy_(g)
        leaves = [sx.detach().requires_grad_(True), sg.detach().requires_grad_(True)]
        h, ht = gated_recurrence(*leaves, initial_state=h0, output_final_state=True)
        # (not against a call on contiguous tensors, whose steps may be others: two roundings of what differs in fp32 may be a whole step apart)
        r = O.recurrence(x.view(-1, D), g.view(-1, D), h0, O.dense_bounds(B, T), dh.view(-1, D))
        close('h', h.detach().reshape(-1, D), r['h'], r['h_off'])
        close('ht', ht.detach(), r['ht'], r['ht_off'])
        for name, t in zip(('dx', 'dg'), torch.autograd.grad(h, leaves, dh)):
            close(name, t.reshape(-1, D), r[name], r[name + '_off'])
    # neither slices nor rows: what cannot be read in place is copied
    x, g, h0, _, _ = make(4, 60, 32, 4, F, F, True, seed=6)
    for view in (lambda t: t.transpose(0, 1).contiguous().transpose(0, 1), lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)):
        assert torch.equal(gated_recurrence(view(x), view(g), h0)[0], gated_recurrence(x, g, h0)[0])
    one = x[:, :, :1]
    assert torch.equal(gated_recurrence(one.expand(4, 60, 32), g, h0)[0], gated_recurrence(one.expand(4, 60, 32).contiguous(), g, h0)[0])


def test_gates_at_their_ends():
    """Minus infinity forgets, whatever was before; zero keeps; a state, gate or input that is not finite stays with its channel and with
    what follows (in the gradient: precedes) it."""
    from b200gdn import gated_recurrence
    for T, D in ((200, 64), (1500, 32), (40, 5)):
        x, g, h0, dh, dht = make(1, T, D, 1, F, F, True, seed=7)
        g[0, T // 2] = -float('inf')
        g[0, T // 2 + 3:, :2] = 0.0
        run_and_check(x, g, h0, dh, dht, [(0, T)])
        for gt in (BF, F):
            xb, gb = x.to(gt), g.to(gt)
            clean, _ = gated_recurrence(xb, gb, h0)
            at = T // 3
            bad = xb.clone()
            bad[0, at, 1] = float('nan')
            leaf = gb.clone().requires_grad_(True)
            h, _ = gated_recurrence(bad, leaf, h0)
            assert torch.isnan(h[0, at:T // 2, 1]).all() and torch.equal(h[0, :at].detach(), clean[0, :at])
            keep = [c for c in range(D) if c != 1]
            assert torch.equal(h[0, :, keep].detach(), clean[0, :, keep])
            dg, = torch.autograd.grad(h, leaf, torch.ones_like(h))
            assert torch.isfinite(dg[0, :, keep]).all() and torch.isfinite(dg[0, :at, 1]).all()


def test_gradient_of_differences():
    """In fp32 along a direction, (f(z + e d) - f(z - e d)) / 2e with e = 2^-7: f is smooth on the scale of a gate of one, the third
    derivative leaves about e^2 / 6 x (a few tokens' decay)^2, rounding 2^-24 / e x sqrt(terms): 2e-3 of the sum of absolute terms' root."""
    from b200gdn import gated_recurrence
    x, g, h0, dh, dht = make(2, 150, 40, 2, F, F, True, seed=8, fast=True)
    d = [torch.randn_like(t) for t in (x, g, h0)]
    leaves = [t.clone().requires_grad_(True) for t in (x, g, h0)]

    def f(e):
        h, ht = gated_recurrence(*(t + e * v for t, v in zip((x, g, h0), d)), output_final_state=True)
        return (h.double() * dh).sum() + (ht.double() * dht).sum()
    h, ht = gated_recurrence(*leaves, output_final_state=True)
    got = torch.autograd.grad([h, ht], leaves, [dh, dht])
    along = sum((a.double() * b).sum() for a, b in zip(got, d))
    e = 2.0 ** -7
    scale = sum((a.double() * b).square().sum() for a, b in zip(got, d)).sqrt()
    assert abs((f(e) - f(-e)) / (2 * e) - along) < 2e-3 * scale + 1e-3 * abs(along)


def test_states_carried_from_call_to_call():
    """A sequence in pieces (one token, few, many), the state updated in place, against one call over all of it."""
    from b200gdn import gated_recurrence
    for D, dtype in ((64, BF), (33, F)):
        x, g, h0, _, _ = make(3, 400, D, 3, dtype, dtype, True, seed=9)
        want, want_t = gated_recurrence(x, g, h0, output_final_state=True)
        r = O.recurrence(x.reshape(-1, D), g.reshape(-1, D), h0, O.dense_bounds(3, 400))
        state, at, parts = h0.clone(), 0, []
        for n in (1, 1, 5, 130, 1, 262):
            h, s = gated_recurrence(x[:, at:at + n], g[:, at:at + n], state, output_final_state=True, inplace_state=True)
            assert s is state or s.data_ptr() == state.data_ptr()
            parts.append(h)
            at += n
        # (each piece hands its state on in fp32: the same bound as for the sequence in one)
        close('h', torch.cat(parts, 1).reshape(-1, D), r['h'], r['h_off'])
        close('ht', state, r['ht'], r['ht_off'])
        close('ht', want_t, r['ht'], r['ht_off'])


def test_one_token_a_sequence_as_packed_and_as_a_batch():
    from b200gdn import gated_recurrence
    x, g, h0, _, _ = make(70, 1, 48, 70, BF, BF, True, seed=10)
    a = gated_recurrence(x, g, h0, output_final_state=True)
    cu = torch.arange(71, dtype=torch.int32, device='cuda')
    b = gated_recurrence(x.view(1, 70, 48), g.view(1, 70, 48), h0, output_final_state=True, cu_seqlens=cu)
    assert torch.equal(a[0].view(70, 48), b[0].view(70, 48)) and torch.equal(a[1], b[1])


def test_no_tokens():
    from b200gdn import gated_recurrence
    h0 = torch.randn(2, 8, device='cuda', requires_grad=True)
    x = torch.zeros(2, 0, 8, device='cuda', requires_grad=True)
    h, ht = gated_recurrence(x, x, h0, output_final_state=True)
    assert h.shape == x.shape and torch.equal(ht, h0)
    d, = torch.autograd.grad(ht, h0, torch.full_like(ht, 3.0))
    assert (d == 3).all()
    assert (gated_recurrence(x.detach(), x.detach(), output_final_state=True)[1] == 0).all()
    assert gated_recurrence(torch.zeros(0, 4, 8, device='cuda'), torch.zeros(0, 4, 8, device='cuda'))[0].shape == (0, 4, 8)


def test_types_of_gates_and_states():
    from b200gdn import gated_recurrence
    x, g, h0, dh, _ = make(2, 20, 16, 2, BF, F, True, seed=11)
    for gt in (HF, torch.float64):   # neither the type of x nor fp32
        leaf = g.to(gt).requires_grad_(True)
        h, _ = gated_recurrence(x, leaf, h0.half())
        assert torch.equal(h.detach(), gated_recurrence(x, leaf.detach().float(), h0.half().float())[0])
        assert torch.autograd.grad(h, leaf, dh)[0].dtype == gt
    s = h0.bfloat16().requires_grad_(True)
    h, ht = gated_recurrence(x, g, s, output_final_state=True)
    assert ht.dtype == F and torch.autograd.grad(h, s, dh)[0].dtype == BF
    for need in range(3):   # one of the three alone
        leaves = [t.clone().requires_grad_(i == need) for i, t in enumerate((x, g, h0))]
        h, _ = gated_recurrence(*leaves)
        every = [t.clone().requires_grad_(True) for t in (x, g, h0)]
        assert torch.equal(torch.autograd.grad(h, leaves[need], dh)[0], torch.autograd.grad(gated_recurrence(*every)[0], every[need], dh)[0])


def test_streams_and_graphs():
    """On another stream, and captured: forward, backward and a decoding step replayed on new data."""
    from b200gdn import gated_recurrence
    args = [make(2, 300, 96, 2, BF, BF, True, seed=s) for s in (12, 13)]
    cu = torch.tensor([0, 100, 100, 600], dtype=torch.int32, device='cuda')
    args3 = [make(1, 600, 96, 3, BF, BF, True, seed=s) for s in (14, 15)]

    def both(x, g, h0, dh, dht, cu):
        x, g, h0 = (t.detach().requires_grad_(True) for t in (x, g, h0))
        h, ht = gated_recurrence(x, g, h0, output_final_state=True, cu_seqlens=cu)
        return [h.detach(), ht.detach(), *torch.autograd.grad([h, ht], [x, g, h0], [dh, dht])]
    for pair, c in ((args, None), (args3, cu)):
        want = [both(*a, c) for a in pair]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = both(*pair[0], c)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(p, q) for p, q in zip(got, want[0]))
        held = [t.clone() for t in pair[0]]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = both(*held, c)
        for a, w in ((pair[1], want[1]), (pair[0], want[0])):
            for t, n in zip(held, a):
                t.copy_(n)
            graph.replay()
            assert all(torch.equal(p, q) for p, q in zip(out, w))
    x, g, h0, _, _ = make(4, 1, 64, 4, BF, BF, True, seed=16)
    state, graph = h0.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = gated_recurrence(x, g, state, output_final_state=True, inplace_state=True)
    ref = h0.clone()
    for _ in range(3):
        graph.replay()
        want, _ = gated_recurrence(x, g, ref, output_final_state=True, inplace_state=True)
        assert torch.equal(out, want) and torch.equal(state, ref)


def test_a_trace_replays_the_operator():
    from b200gdn import gated_recurrence
    x, g, _, _, _ = make(2, 70, 64, 2, F, F, False, seed=17)
    traced = torch.jit.trace(lambda a, b: gated_recurrence(a, b)[0], (x, g))
    y, k, _, _, _ = make(3, 130, 64, 3, F, F, False, seed=18)
    assert torch.equal(traced(y, k), gated_recurrence(y, k)[0])


def test_a_long_sequence_of_many_rows():
    """Offsets beyond 2^31 elements: the last channels' and rows' results are those of a short call from the state before them."""
    from b200gdn import gated_recurrence
    T, D = 300000, 8192
    x = torch.full((1, T, D), 0.5, dtype=BF, device='cuda')
    g = torch.full((1, T, D), -0.125, dtype=BF, device='cuda')
    tail = torch.randn(1, 100, D, device='cuda').to(BF)
    x[:, -100:] = tail
    h, ht = gated_recurrence(x, g, output_final_state=True)
    before = torch.full((1, D), 0.5 / (1 - 2.718281828459045 ** -0.125), device='cuda')   # (where the first tokens' share is below any digit)
    r = O.recurrence(tail[0], g[0, -100:], before, [(0, 100)])
    # the state before the tail is a fixed point, reached up to 16 U x its size / (1 - decay)
    off = r['h_off'] + 16 * O.U * before.double() / (1 - 2.718281828459045 ** -0.125)
    close('h', h[0, -100:], r['h'], off)
    close('ht', ht, r['ht'], off[-1:])


def test_refusals():
    from b200gdn import B200GDNError, gated_recurrence
    x = torch.zeros(2, 3, 8, device='cuda')
    with pytest.raises(B200GDNError, match='not supported'):
        gated_recurrence(x.double(), x.double())
    with pytest.raises(B200GDNError, match='batch, tokens, channels'):
        gated_recurrence(x[0], x[0])
    with pytest.raises(B200GDNError, match='shape of x'):
        gated_recurrence(x, x[:, :2])
    with pytest.raises(B200GDNError, match='shape of x'):
        gated_recurrence(x, x.long())
    with pytest.raises(B200GDNError, match='is on cpu'):
        gated_recurrence(x, x.cpu())
    for s in (x[0, :1], x[:, 0, :7], x):
        with pytest.raises(B200GDNError, match='a state a sequence'):
            gated_recurrence(x, x, s)
    with pytest.raises(B200GDNError, match='fp32'):
        gated_recurrence(x, x, x[:, 0].half(), output_final_state=True, inplace_state=True)
    with pytest.raises(B200GDNError, match='fp32'):
        gated_recurrence(x, x, None, output_final_state=True, inplace_state=True)
    with pytest.raises(ValueError, match='output_final_state'):
        gated_recurrence(x, x, x[:, 0].contiguous(), inplace_state=True)
    leaf = x.clone().requires_grad_(True)
    with pytest.raises(B200GDNError, match='gradients'):
        gated_recurrence(leaf, x, x[:, 0].contiguous(), output_final_state=True, inplace_state=True)
    with pytest.raises(ValueError, match='batch size'):
        gated_recurrence(x, x, cu_seqlens=torch.tensor([0, 3], device='cuda'))
    with pytest.raises(ValueError, match='outside'):
        gated_recurrence(x[:1], x[:1], cu_seqlens=torch.tensor([0, 4], device='cuda'))
    dx, = torch.autograd.grad(gated_recurrence(leaf, x)[0].square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match='no second derivative'):
        dx.sum().backward()


def _token_by_token(x, g, h0, dh, dht):
    """h, the last state, dx, dg and dh0 of sequences [B, T, D], in 64 bits and in the definition's order."""
    a = torch.exp(g.double())
    x, dh, h, u = x.double(), dh.double(), h0.double(), dht.double()
    hs, before, dx, dg = [], [], [None] * x.shape[1], [None] * x.shape[1]
    for t in range(x.shape[1]):
        before.append(h)
        h = a[:, t] * h + x[:, t]
        hs.append(h)
    for t in range(x.shape[1] - 1, -1, -1):
        dx[t] = dh[:, t] + u
        dg[t] = dx[t] * (a[:, t] * before[t])
        u = a[:, t] * dx[t]
    return torch.stack(hs, 1), h, torch.stack(dx, 1), torch.stack(dg, 1), u


@pytest.mark.parametrize('B,T,D', [(1, 7, 32), (2, 100, 64), (1, 700, 64), (1, 700, 35), (1, 5000, 64), (8, 400, 1280), (8, 400, 1283), (2, 300, 1280)])
@pytest.mark.parametrize('dtype,gtype', [(BF, BF), (HF, F), (F, F)])
def test_a_state_that_is_infinite_stays_so(B, T, D, dtype, gtype):
    """While no decay is zero, however far their product over many tokens falls below fp32's range: where the definition has an infinity or NaN, there
    it is, of the same sign, and nowhere else."""
    from b200gdn import gated_recurrence
    inf = float('inf')
    for gate in (-1.5, -12.0):   # the product leaves the range over 64 tokens, over eight
        x, _, h0, dh, dht = make(B, T, D, B, dtype, gtype, True, seed=T)
        g = torch.full((B, T, D), gate, device='cuda').to(gtype)
        h0[:, 0], h0[:, 1], x[:, T // 3, 2], x[:, T // 4, 3], x[:, T // 2, 3] = inf, -inf, inf, inf, -inf
        x[:, 2, 4], g[:, T // 2, 4] = -inf, -inf          # a decay of zero: NaN from there on
        dht[:, 5], dht[:, 6], dh[:, T // 2, 7], dh[:, T - 1, 8], dh[:, T // 2, 8] = inf, -inf, inf, -inf, inf
        dh[:, T // 2, 9], g[:, T // 3, 9] = inf, -inf
        leaves = [t.clone().requires_grad_(True) for t in (x, g, h0)]
        h, ht = gated_recurrence(*leaves, output_final_state=True)
        got = [h.detach(), ht.detach(), *torch.autograd.grad([h, ht], leaves, [dh, dht])]
        for name, p, q in zip(('h', 'ht', 'dx', 'dg', 'dh0'), got, _token_by_token(x, g, h0, dh, dht)):
            p = p.double()
            assert torch.equal(torch.isnan(p), torch.isnan(q)), (name, gate)
            assert torch.equal(p[torch.isinf(p)], q[torch.isinf(p)]) and torch.equal(torch.isinf(p), torch.isinf(q)), (name, gate)


def side_by_side(t):
    """[B, T, ...] as [T, B ...]: sequences of one length as channels of one, which the oracle walks in T steps"""
    return t.transpose(0, 1).reshape(t.shape[1], -1)


def run_side_by_side(x, g, h0, dh, dht):
    from b200gdn import gated_recurrence
    leaves = [t if t is None else t.clone().requires_grad_(True) for t in (x, g, h0)]
    h, ht = gated_recurrence(*leaves, output_final_state=True)
    r = O.recurrence(side_by_side(x), side_by_side(g), None if h0 is None else h0.reshape(1, -1), [(0, x.shape[1])], side_by_side(dh), dht.reshape(1, -1))
    got = torch.autograd.grad([h, ht], [t for t in leaves if t is not None], [dh, dht])
    for name, t in (('h', h.detach()), ('dx', got[0]), ('dg', got[1])):
        close(name, side_by_side(t), r[name], r[name + '_off'])
    close('ht', ht.detach().reshape(1, -1), r['ht'], r['ht_off'])
    if h0 is not None:
        close('dh0', got[2].reshape(1, -1), r['dh0'], r['dh0_off'])


@pytest.mark.parametrize('B,T,D', [(8, 700, 1280), (8, 641, 1290), (8, 700, 1283), (5, 1300, 2056), (1, 6000, 64), (1, 6100, 33), (3, 3000, 130)])
@pytest.mark.parametrize('dtype,gtype', [(BF, BF), (BF, F), (HF, HF), (F, F)])
def test_many_steps(B, T, D, dtype, gtype):
    """More pieces of work than SMs, where a CTA has its sequence alone and walks it in many steps (by TMA, by pairs, by single elements); and
    few channels in clusters, three and more steps of the largest."""
    for h0 in (True, False):
        run_side_by_side(*make(B, T, D, B, dtype, gtype, h0, seed=T))


@pytest.mark.parametrize('B,T,D,most', [(2, 40, 64, 0.5), (2, 1, 8, 3.0), (1, 3000, 64, 0.03), (1, 2500, 35, 0.03), (8, 400, 1280, 0.1), (3, 7, 5, 2.0)])
@pytest.mark.parametrize('dtype,gtype', [(BF, BF), (BF, F), (F, F)])
def test_gates_above_zero(B, T, D, most, dtype, gtype):
    """States that grow, by up to e^45 over a sequence, beside channels that forget."""
    x, _, h0, dh, dht = make(B, T, D, B, dtype, gtype, True, seed=D)
    g = most * torch.rand(B, T, D, device='cuda')
    g[..., 1::3] *= -1
    g[..., 2::3] -= most / 2
    run_side_by_side(x, g.to(gtype), h0, dh, dht)


def test_the_gradient_of_a_long_sequence_of_many_rows():
    """Offsets beyond 2^31 elements, backward: the last rows' gradients are those of a short call from the state before them."""
    from b200gdn import gated_recurrence
    T, D, n = 300000, 8192, 200
    x = torch.full((1, T, D), 0.5, dtype=BF, device='cuda')
    g = torch.full((1, T, D), -0.125, dtype=BF, device='cuda')
    dh = torch.zeros(1, T, D, dtype=BF, device='cuda')
    for t in (x, dh):
        t[:, -n:] = torch.randn(1, n, D, device='cuda').to(BF)
    dht = torch.randn(1, D, device='cuda')
    leaves = [x.requires_grad_(True), g.requires_grad_(True)]
    h, ht = gated_recurrence(*leaves, output_final_state=True)
    dx, dg = torch.autograd.grad([h, ht], leaves, [dh, dht])
    before = torch.full((1, D), 0.5 / (1 - 2.718281828459045 ** -0.125), device='cuda')
    r = O.recurrence(x.detach()[0, -n:], g.detach()[0, -n:], before, [(0, n)], dh[0, -n:], dht)
    close('dx', dx[0, -n:], r['dx'], r['dx_off'])
    # (the state before the tail is off by up to 16 U x its size / (1 - decay), and what is left of it multiplies dx)
    left = torch.exp(-0.125 * torch.arange(1, n + 1, device='cuda').double())[:, None]
    off = 16 * O.U * before.double() / (1 - 2.718281828459045 ** -0.125)
    close('dg', dg[0, -n:], r['dg'], r['dg_off'] + r['dx'].abs() * left * off)
    assert (dx[0, :1000] == 0).all() and (dg[0, :1000] == 0).all()   # what is left so far ahead is below any digit
