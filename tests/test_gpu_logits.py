"""Log probabilities and the distillation loss on the GPU against the 64-bit restatements.

Tolerances, from the arithmetic.  Log probabilities in 32 bits: a difference of two logits and its product with 1/T (2 units of
2^-24 of the difference), the logarithm of a sum whose terms are off by 2^-22 (exponential) plus 2^-24 of their exponent, and
whose additions run in chains of some hundred terms, whose errors average out: 2^-20 is allowed.  The entropy and a row's loss are
means of such.
Gradients: rounded once to the logits' type (a unit in the last place is allowed), made of terms (`dx_size`) each off by that of a
probability: 2^-20 and 2^-22 of the exponent, which is at most 100 where the term counts: 2^-15."""
import math

import pytest
import torch

from oracle import head_oracle as H

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
EPS = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -23}
TINY = {torch.bfloat16: 1e-37, torch.float16: 2.0 ** -24, torch.float32: 1e-37}
VOCABS = [1, 2, 3, 8, 17, 64, 100, 257, 1000, 1023, 4097, 8192, 20000, 32000, 50001, 65537, 131072]


def close_lp(name, got, want):
    assert got.dtype == torch.float32
    same = got.double() == want                       # infinities
    fine = (got.double() - want).abs() <= 2.0 ** -20 + 2.0 ** -22 * want.abs()
    assert (same | fine).all(), f'{name}: off by {torch.where(same, 0.0, (got.double() - want).abs()).max().item():.3g}'


def close_grad(name, got, want, size):
    limit = EPS[got.dtype] * want.abs() + 2.0 ** -15 * size + TINY[got.dtype]
    off = (got.double() - want).abs() / limit
    assert torch.isfinite(got).all(), name
    assert off.max() <= 1.0, f'{name}: {off.max().item():.2f} of what is allowed'


def gen(seed=0):
    return torch.Generator(device='cuda').manual_seed(seed)


def logits_of(n, v, dtype, seed=0, spread=3.0):
    return (torch.randn(n, v, device='cuda', generator=gen(seed)) * spread).to(dtype)


def tokens_of(n, v, seed=0, some=True):
    t = torch.randint(0, v, (n,), device='cuda', generator=gen(seed + 77))
    if some and n > 2:
        t[1] = -100
        t[2] = v          # past the end: asks for nothing
    return t


def check_logprobs(x, tokens, k, temperature=1.0, upstream=True):
    """x: the tensor as it is handed over, any strides."""
    from b200gdn import token_logprobs
    flat = x.detach().reshape(-1, x.shape[-1])
    leaf = x.detach().requires_grad_(True) if upstream else x
    r = token_logprobs(leaf, tokens, top_k=k, temperature=temperature)
    values, ups = [r.logprobs, r.entropy], []
    if k:
        values.append(r.top_logprobs)
    if upstream:
        ups = [torch.randn(v.shape, device='cuda', generator=gen(5 + i)) for i, v in enumerate(values)]
    want = H.logprobs(flat, tokens.reshape(-1), k, temperature, *(u.reshape(-1, *u.shape[x.dim() - 1:]) for u in ups))
    close_lp('logprobs', r.logprobs.detach().reshape(-1), want['logprobs'])
    close_lp('entropy', r.entropy.detach().reshape(-1), want['entropy'])
    if k:
        assert r.top_ids.dtype == torch.int64 and r.top_ids.shape == (*x.shape[:-1], k)
        assert torch.equal(r.top_ids.reshape(-1, k), want['top_ids'])
        close_lp('top_logprobs', r.top_logprobs.detach().reshape(-1, k), want['top_logprobs'])
    if upstream:
        dx, = torch.autograd.grad(values, leaf, ups)
        assert dx.shape == x.shape and dx.dtype == x.dtype
        close_grad('dlogits', dx.reshape(flat.shape), want['dx'], want['dx_size'])
        with torch.no_grad():
            again = token_logprobs(x, tokens, top_k=k, temperature=temperature)
        assert all(torch.equal(p, q) for p, q in zip(again, r) if p is not None)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('V', VOCABS)
def test_logprobs(V, dtype):
    for i, (n, k, temperature) in enumerate([(1, 20, 1.0), (7, 1, 0.6), (33, 128, 2.0), (200 if V <= 65537 else 20, 0, 1.0), (300 if V < 9000 else 5, 64, 1.0)]):
        check_logprobs(logits_of(n, V, dtype, i), tokens_of(n, V, i), min(k, V), temperature)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('V', [300, 5003, 40000])
@pytest.mark.parametrize('kind', ['equal', 'few', 'rising', 'falling', 'blocks', 'zeros'])
def test_top_entries_in_any_order(kind, V, dtype):
    """Ties all over, sorted rows, the largest entries side by side; the zeros of both signs are equal."""
    n = 6
    x = torch.full((n, V), 1.5, device='cuda')
    if kind == 'few':
        x = torch.randint(0, 4, (n, V), device='cuda', generator=gen()).float()
    elif kind in ('rising', 'falling'):
        x = torch.linspace(-20, 20, V, device='cuda').expand(n, V) + torch.arange(n, device='cuda')[:, None]
        x = x if kind == 'rising' else -x
    elif kind == 'blocks':
        x = torch.randn(n, V, device='cuda', generator=gen())
        for i in range(n):
            x[i, 37 * i:37 * i + 200] += 30
    elif kind == 'zeros':
        x = torch.where(torch.rand(n, V, device='cuda', generator=gen()) < 0.5, 0.0, -0.0)
    for k in (1, 2, 31, 128):
        check_logprobs(x.to(dtype), tokens_of(n, V), k, upstream=False)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('k', [1, 20, 128])
def test_top_entries_that_lie_together(k, dtype):
    """Thousands of entries above all others, at the places that few lanes of the kernels hold; few entries that are not masked."""
    from b200gdn import token_logprobs
    V = 131072
    at = torch.arange(V, device='cuda')
    x = torch.randn(4, V, device='cuda', generator=gen())
    x[:, at // (4 if dtype == torch.float32 else 8) % 32 < 2] += 20
    x[1] = torch.where(torch.rand(V, device='cuda', generator=gen(1)) < 1e-4, x[1], -math.inf)
    x[2] = torch.where(at < 3, x[2], torch.finfo(dtype).min)
    x[3] = torch.where(at >= V - 300, 2.0, -math.inf)
    check_logprobs(x.to(dtype), tokens_of(4, V), k, upstream=False)
    for temperature in (1e-4, 3e4):
        r, want = token_logprobs(x.to(dtype), top_k=k, temperature=temperature), H.logprobs(x.to(dtype), tokens_of(4, V), k, temperature)
        assert torch.equal(r.top_ids, want['top_ids'])
        close_lp('entropy', r.entropy, want['entropy'])


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('V', [40, 1003, 33000])
def test_masked_entries(V, dtype):
    """Minus infinity and the type's lowest value in masked places, rows with little or nothing left, a token that is masked."""
    x = logits_of(12, V, dtype)
    x[torch.rand(12, V, device='cuda', generator=gen(1)) < 0.5] = -math.inf
    x[1] = -math.inf                                   # nothing
    x[2] = -math.inf
    x[2, V // 2] = 3.0                                 # one entry
    x[3] = torch.finfo(dtype).min                      # all at the lowest value: equal
    x[4] = torch.finfo(dtype).min
    x[4, 5:9] = 1.0
    x[5, :] = torch.finfo(dtype).min / 2
    x[5, 7] = torch.finfo(dtype).min
    x[6, 3] = torch.finfo(dtype).max                   # all the others are nothing
    tokens = torch.full((12,), 5, device='cuda')
    tokens[2] = V // 2
    x[7, 5] = -math.inf
    for k in (0, 20):
        check_logprobs(x, tokens, k)
    from b200gdn import token_logprobs
    r = token_logprobs(x, tokens, top_k=20)
    assert r.entropy[1] == 0 and (r.logprobs[[1, 7]] == -math.inf).all() and (r.top_logprobs[1] == -math.inf).all()
    assert torch.equal(r.top_ids[1], torch.arange(20, device='cuda'))


@pytest.mark.parametrize('dtype', DTYPES)
def test_infinity_and_nan(dtype):
    """What the formulas give: a row with infinity or NaN has no number for a result.  Its neighbours have theirs, and the
    indices stay inside the vocabulary."""
    from b200gdn import token_logprobs
    for V in (50, 30011):
        x = logits_of(5, V, dtype)
        clean = token_logprobs(x, tokens_of(5, V, some=False), top_k=5)
        x[1, 7] = math.inf
        x[3, V - 1] = math.nan
        leaf = x.requires_grad_(True)
        r = token_logprobs(leaf, tokens_of(5, V, some=False), top_k=5)
        for i in range(5):
            bad = i in (1, 3)
            assert bool(r.logprobs[i].isnan()) == bad and bool(r.entropy[i].isnan()) == bad
            if not bad:
                assert r.logprobs[i] == clean.logprobs[i] and torch.equal(r.top_ids[i], clean.top_ids[i])
        assert r.top_ids[1, 0] == 7 and r.top_ids[3, 0] == V - 1 and ((r.top_ids >= 0) & (r.top_ids < V)).all()
        dx, = torch.autograd.grad(r.logprobs.sum(), leaf)
        assert dx[[1, 3]].isnan().any(-1).all() and dx[[0, 2, 4]].isfinite().all()


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('V', [97, 1000, 30001])
def test_logprobs_of_slices(V, dtype):
    """Logits where they lie: all but the last token of each sequence, a padded vocabulary, off every boundary, other orders."""
    B, T = 3, 5
    whole = logits_of(B * (T + 1) * 2, V + 11, dtype).view(B, T + 1, 2, V + 11)
    for x in (whole[:, :-1, 0, :V], whole[:, 1:, 1, 3:V + 3], whole[0, :, 0, 1:V + 1], whole[:, 0, :, 11:], whole[:, :-1, :, 2:V + 2],
              whole.transpose(0, 1)[..., :V], whole[0, 0, 0, 5:5 + V], whole[:, 0, 0, :V].expand(4, B, V)):
        check_logprobs(x, tokens_of(x[..., 0].numel(), V).view(x.shape[:-1]), min(20, V))
    check_logprobs(whole[0, :, 0, :V * 1].transpose(0, 1).contiguous().transpose(0, 1), tokens_of(T + 1, V), 3)


def test_logprobs_options():
    from b200gdn import token_logprobs
    x, t = logits_of(9, 5000, torch.bfloat16), tokens_of(9, 5000)
    full = token_logprobs(x, t, top_k=4)
    part = token_logprobs(x, t.int(), return_entropy=False)
    assert part.entropy is None and part.top_ids is None and torch.equal(part.logprobs, full.logprobs)
    part = token_logprobs(x, top_k=4)
    assert part.logprobs is None and torch.equal(part.top_ids, full.top_ids) and torch.equal(part.entropy, full.entropy)
    # any part of the results may be used
    want = H.logprobs(x, t, 4, 1.0, None, torch.ones(9, device='cuda'))
    leaf = x.clone().requires_grad_(True)
    r = token_logprobs(leaf, t, top_k=4)
    close_grad('entropy alone', torch.autograd.grad(r.entropy.sum(), leaf, retain_graph=True)[0], want['dx'], want['dx_size'])
    up = torch.randn(9, 8, device='cuda')[:, ::2]
    want = H.logprobs(x, t, 4, 1.0, None, None, up)
    close_grad('top alone', torch.autograd.grad(r.top_logprobs, leaf, up)[0], want['dx'], want['dx_size'])
    for empty in (token_logprobs(x[:0], t[:0], top_k=2), token_logprobs(x[:0].float().requires_grad_(True), t[:0], top_k=2)):
        assert empty.logprobs.shape == (0,) and empty.top_ids.shape == (0, 2)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_long_rows(dtype):
    """Rows of millions of entries: more spans than a warp joins in one go, more groups than the top entries are sought by."""
    V = 4_500_001
    x = logits_of(2, V, dtype)
    check_logprobs(x, torch.tensor([V - 1, 7], device='cuda'), 20)
    t, ids = lists_of(2, V, 16, absent=False)
    check_distill(x, t, ids, 1.0, True, ('sum',))


def test_logprobs_past_32_bits():
    """Offsets of more than 2^31 elements; the rows at the end are the same as alone."""
    from b200gdn import token_logprobs
    n, v = 16500, 131072
    x = torch.zeros(n, v, dtype=torch.bfloat16, device='cuda')
    x[-4:] = logits_of(4, v, torch.bfloat16)
    t = torch.full((n,), 3, device='cuda')
    leaf = x.requires_grad_(True)
    r = token_logprobs(leaf, t, top_k=3)
    alone_leaf = x[-4:].detach().clone().requires_grad_(True)
    alone = token_logprobs(alone_leaf, t[-4:], top_k=3)
    assert torch.equal(r.logprobs[-4:], alone.logprobs) and torch.equal(r.top_ids[-4:], alone.top_ids)
    dx, = torch.autograd.grad(r.logprobs.sum() + r.entropy.sum(), leaf)
    want, = torch.autograd.grad(alone.logprobs.sum() + alone.entropy.sum(), alone_leaf)
    assert torch.equal(dx[-4:], want)
    close_lp('equal logits', r.logprobs[:5].detach(), torch.full((5,), -math.log(v), dtype=torch.float64, device='cuda'))


# ---- distillation --------------------------------------------------------------------------------------------------
def lists_of(n, v, k, seed=0, dtype=torch.float32, absent=True):
    ids = torch.rand(n, v, device='cuda', generator=gen(seed)).argsort(-1)[:, :k]
    t = torch.log_softmax(torch.randn(n, k + 1, device='cuda', generator=gen(seed + 1)) * 2, -1)[:, :k].contiguous().to(dtype)
    if absent and n > 5:
        ids[0] = -1                     # no teacher
        ids[1, k // 2:] = -100          # a short list (none for one entry)
        ids[2, 0] = v                   # past the end
        t[3, 0] = -math.inf
        t[4] = -math.inf
        if k > 3:
            ids[5, 3] = ids[5, 1]       # an entry given twice
    return t, ids


def check_distill(x, t, ids, temperature=1.0, bucket=False, reductions=('mean', 'sum', 'none')):
    from b200gdn import topk_distill_loss
    flat = x.detach().reshape(-1, x.shape[-1])
    want = H.distill(flat, t.reshape(-1, t.shape[-1]), ids.reshape(-1, t.shape[-1]), temperature, bucket)
    options = dict(temperature=temperature, remainder='bucket' if bucket else 'renormalize')
    for red in reductions:
        leaf = x.detach().requires_grad_(True)
        loss = topk_distill_loss(leaf, t, ids, reduction=red, **options)
        total, factor = H.reduce_loss(want['rows'], want['counted'], red)
        # a row's loss is a mean of log probabilities (and their like), as far off as those
        limit = torch.where(want['counted'], 2.0 ** -20 + 2.0 ** -22 * want['rows_size'], 0.0)
        if red != 'none':
            limit = limit.sum() * factor + 2.0 ** -22 * want['rows'].abs().sum() * factor
        got = loss.detach().double().reshape(total.shape)
        assert ((got == total) | ((got - total).abs() <= limit)).all(), (red, (got - total).abs().max())
        with torch.no_grad():
            again = topk_distill_loss(x, t, ids, reduction=red, **options)
        assert ((again == loss.detach()) | ((again - loss.detach()).abs() <= 2 * limit.view(again.shape))).all()
        if red == 'none':
            up = torch.randn(loss.shape, device='cuda', generator=gen(9))
            dx, = torch.autograd.grad(loss, leaf, up)
            close_grad('dlogits', dx.reshape(flat.shape), want['dx'] * up.reshape(-1, 1), want['dx_size'] * up.reshape(-1, 1).abs())
            continue
        dx, = torch.autograd.grad(loss, leaf, retain_graph=True)
        close_grad('dlogits', dx.reshape(flat.shape), want['dx'] * factor, want['dx_size'] * factor)
        kept = dx.clone()
        scaled, = torch.autograd.grad(loss, leaf, torch.tensor(2.5, device='cuda'), retain_graph=True)   # a second time, another factor
        close_grad('dlogits', scaled.reshape(flat.shape), 2.5 * factor * want['dx'], 2.5 * factor * want['dx_size'])
        assert torch.equal(dx, kept)
        leaf2 = x.detach().requires_grad_(True)                                                           # a first time with a factor
        dx, = torch.autograd.grad(topk_distill_loss(leaf2, t, ids, reduction=red, **options) * -0.3, leaf2)
        close_grad('dlogits', dx.reshape(flat.shape), -0.3 * factor * want['dx'], 0.3 * factor * want['dx_size'])


@pytest.mark.parametrize('bucket', [False, True])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('V', VOCABS)
def test_distill(V, dtype, bucket):
    for i, (n, k, temperature) in enumerate([(1, 20, 1.0), (7, 1, 0.6), (33, 128, 2.0), (90 if V <= 65537 else 20, 64, 1.0), (9, 256, 1.0)]):
        t, ids = lists_of(n, V, min(k, V), i, [torch.float32, torch.bfloat16][i % 2])
        check_distill(logits_of(n, V, dtype, i), t, ids.int() if i == 1 else ids, temperature, bucket)


@pytest.mark.parametrize('bucket', [False, True])
def test_distill_fp16_and_slices(bucket):
    B, T, V = 3, 4, 5003
    whole = logits_of(B * (T + 1), V + 9, torch.float16).view(B, T + 1, V + 9)
    for x in (whole[:, :-1, :V], whole[:, 1:, 3:V + 3], whole[1, :, 5:V + 5], whole[0, 0, :V], whole.transpose(0, 1)[..., 9:]):
        n = x[..., 0].numel()
        t, ids = lists_of(n, V, 20)
        check_distill(x, t.view(*x.shape[:-1], 20), ids.view(*x.shape[:-1], 20), 1.0, bucket, ('sum', 'none'))


@pytest.mark.parametrize('bucket', [False, True])
@pytest.mark.parametrize('V', [70, 33001])
def test_distill_masked_logits(V, bucket):
    """A student with masked entries (of the type's lowest value on the list: a large but finite loss), a row with nothing left
    (infinite loss, no gradient), all the student's mass on the list."""
    from b200gdn import topk_distill_loss
    n, k = 8, 16
    x = logits_of(n, V, torch.float32)
    t, ids = lists_of(n, V, k, absent=False)
    x[1, ids[1, 3]] = -1e30
    x[2] = -math.inf
    x[2].scatter_(0, ids[2], torch.randn(k, device='cuda'))     # nothing off the list
    x[3] = torch.where(torch.rand(V, device='cuda', generator=gen(4)) < 0.5, -math.inf, x[3])
    x[3].scatter_(0, ids[3], torch.randn(k, device='cuda'))
    x[4] -= 60.0
    x[4].scatter_(0, ids[4], torch.randn(k, device='cuda'))     # next to nothing off the list
    finite = [0, 1, 3, 4, 5, 6, 7] if bucket else list(range(8))
    check_distill(x[finite].contiguous(), t[finite], ids[finite], 1.0, bucket)
    rows = topk_distill_loss(x, t, ids, remainder='bucket' if bucket else 'renormalize', reduction='none')
    assert (rows[2] == math.inf) == bucket
    x[5] = -math.inf
    leaf = x.requires_grad_(True)
    rows = topk_distill_loss(leaf, t, ids, reduction='none')
    dx, = torch.autograd.grad(rows.sum(), leaf)
    assert rows[5] == math.inf and (dx[5] == 0).all() and dx[[0, 3]].isfinite().all()
    got, = torch.autograd.grad(topk_distill_loss(leaf, t, ids, reduction='sum'), leaf)
    assert (got[5] == 0).all() and got[[0, 3]].isfinite().all()


def test_distill_nan_stays_in_its_row():
    from b200gdn import topk_distill_loss
    for V in (64, 40001):
        x = logits_of(6, V, torch.bfloat16)
        x[2, V - 3] = math.nan
        t, ids = lists_of(6, V, 8, absent=False)
        t[4, 1] = math.nan
        leaf = x.requires_grad_(True)
        rows = topk_distill_loss(leaf, t, ids, reduction='none')
        assert rows.isnan().tolist() == [False, False, True, False, True, False]
        dx, = torch.autograd.grad(rows.sum(), leaf)
        assert dx[[0, 1, 3, 5]].isfinite().all() and dx[[2, 4]].isnan().any(-1).all()
        total = topk_distill_loss(leaf, t, ids)
        dx, = torch.autograd.grad(total, leaf)
        assert total.isnan() and dx[[0, 1, 3, 5]].isfinite().all() and dx[[2, 4]].isnan().any(-1).all()


def test_distill_without_rows_that_count():
    from b200gdn import topk_distill_loss
    x = logits_of(5, 700, torch.bfloat16).requires_grad_(True)
    t, ids = lists_of(5, 700, 4, absent=False)
    loss = topk_distill_loss(x, t, torch.full_like(ids, -1))
    assert loss == 0 and (torch.autograd.grad(loss, x)[0] == 0).all()
    none = torch.zeros(0, 700, device='cuda', requires_grad=True)
    for red in ('mean', 'sum', 'none'):
        loss = topk_distill_loss(none, t[:0], ids[:0], reduction=red)
        assert loss.sum() == 0
        loss.sum().backward()
    assert none.grad.shape == (0, 700)


def test_gradients_of_differences():
    """fp32, along a direction d of unit variance with h = 2^-5: the third derivatives of these functions are bounded by a few,
    so the truncation is about h^2 / 6 x 4 = 7e-4 of the directional scale; rounding adds 2^-20 x rows / h."""
    from b200gdn import token_logprobs, topk_distill_loss
    x, tok = logits_of(6, 900, torch.float32, spread=1.0), tokens_of(6, 900)
    t, ids = lists_of(6, 900, 12)
    d, h = torch.randn(6, 900, device='cuda', generator=gen(3)), 2.0 ** -5
    top = H.top_ids(x, 40)

    def scores(v):
        r = token_logprobs(v, tok, top_k=3, temperature=1.5)
        return r.logprobs.sum() + 2 * r.entropy.sum() + r.top_logprobs.sum()
    d.scatter_(1, top, 0.0)     # the top entries stay where they are and nothing overtakes them: a change of order is a kink
    for f in (scores, lambda v: topk_distill_loss(v, t, ids, 1.5, 'bucket', 'sum'), lambda v: topk_distill_loss(v, t, ids, 0.8)):
        leaf = x.clone().requires_grad_(True)
        g, = torch.autograd.grad(f(leaf), leaf)
        want = ((f(x + h * d).double() - f(x - h * d).double()) / (2 * h)).item()
        got = (g.double() * d).sum().item()
        assert abs(got - want) < 2e-3 * (1 + (g.double() * d).norm().item() * 6 + abs(want))


def test_results_do_not_depend_on_the_run():
    from b200gdn import token_logprobs, topk_distill_loss
    x = logits_of(700, 32000, torch.bfloat16).requires_grad_(True)
    t, ids = lists_of(700, 32000, 32)
    first = None
    for _ in range(3):
        r = token_logprobs(x, tokens_of(700, 32000), top_k=16)
        loss = topk_distill_loss(x, t, ids, remainder='bucket')
        now = [*(v.detach() for v in r), loss.detach(), *torch.autograd.grad(loss, x), *torch.autograd.grad(r.logprobs.sum() + r.entropy.sum(), x)]
        first = first or now
        assert all(torch.equal(p, q) for p, q in zip(now, first))


def test_streams_graphs_and_traces():
    from b200gdn import token_logprobs, topk_distill_loss
    x, tok = logits_of(40, 9001, torch.bfloat16), tokens_of(40, 9001)
    t, ids = lists_of(40, 9001, 16)

    def step(v):
        leaf = v.detach().requires_grad_(True)
        r = token_logprobs(leaf, tok, top_k=5)
        loss = topk_distill_loss(leaf, t, ids)
        return [*(o.detach() for o in r), loss.detach(), *torch.autograd.grad(loss + r.logprobs.sum(), leaf)]
    want = step(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            kept = step(x)
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    x.copy_(logits_of(40, 9001, torch.bfloat16, 8))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(kept, step(x)))

    def call(v, tk, tt, ti):
        r = token_logprobs(v, tk, top_k=5)
        return r.logprobs, r.top_ids, topk_distill_loss(v, tt, ti)
    traced = torch.jit.trace(call, (x, tok, t, ids))
    other = logits_of(11, 9001, torch.bfloat16, 3)
    args = (other, tok[:11], t[:11], ids[:11])
    assert all(torch.equal(p, q) for p, q in zip(traced(*args), call(*args)))


def test_refusals():
    from b200gdn import B200GDNError, token_logprobs, topk_distill_loss
    x, tok = logits_of(4, 200, torch.float32), tokens_of(4, 200)
    t, ids = lists_of(4, 200, 3)
    for call, match in [
        (lambda: token_logprobs(x.cpu(), tok), 'CUDA device only'),
        (lambda: token_logprobs(x.double(), tok), 'not supported'),
        (lambda: token_logprobs(x[:, :0], tok), 'without entries'),
        (lambda: token_logprobs(x, tok[:3]), 'another shape'),
        (lambda: token_logprobs(x, tok.float()), 'int32 or int64'),
        (lambda: token_logprobs(x, tok.cpu()), 'is on cpu'),
        (lambda: token_logprobs(x, tok, top_k=129), 'top_k'),
        (lambda: token_logprobs(x[:, :5], tok, top_k=6), 'top_k'),
        (lambda: token_logprobs(x, tok, top_k=-1), 'top_k'),
        (lambda: token_logprobs(x, return_entropy=False), 'nothing is asked'),
        (lambda: topk_distill_loss(x.cpu(), t, ids), 'CUDA device only'),
        (lambda: topk_distill_loss(x, t[:3], ids), 'another shape'),
        (lambda: topk_distill_loss(x, t, ids[:, :2]), 'another shape'),
        (lambda: topk_distill_loss(x, t[:, :0], ids[:, :0]), 'entries a row'),
        (lambda: topk_distill_loss(x, t.expand(100, 4, 3).permute(1, 2, 0).reshape(4, 300), ids.repeat(1, 100)), 'entries a row'),
        (lambda: topk_distill_loss(x, t.double(), ids), 'of type'),
        (lambda: topk_distill_loss(x, t, ids.short()), 'int32 or int64'),
        (lambda: topk_distill_loss(x, t.clone().requires_grad_(True), ids), 'detach'),
    ]:
        with pytest.raises(B200GDNError, match=match):
            call()
    for temperature in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match='temperature'):
            token_logprobs(x, tok, temperature=temperature)
    with pytest.raises(ValueError, match='remainder'):
        topk_distill_loss(x, t, ids, remainder='drop')
    with pytest.raises(ValueError, match='reduction'):
        topk_distill_loss(x, t, ids, reduction='batchmean')
    leaf = x.clone().requires_grad_(True)
    for value in (token_logprobs(leaf, tok).logprobs.square().sum(), topk_distill_loss(leaf, t, ids)):
        dx, = torch.autograd.grad(value, leaf, create_graph=True)
        with pytest.raises(RuntimeError, match='no second derivative'):
            dx.sum().backward()


def test_forward_mode_tangents_are_refused():
    import torch.autograd.forward_ad as fw
    from b200gdn import layer_norm, token_logprobs, topk_distill_loss
    x, tok = logits_of(4, 64, torch.float32), tokens_of(4, 64)
    t, ids = lists_of(4, 64, 3)
    with fw.dual_level():
        dual = fw.make_dual(x, torch.ones_like(x))
        for call in (lambda: token_logprobs(dual, tok), lambda: topk_distill_loss(dual, t, ids), lambda: layer_norm(dual)):
            with pytest.raises((NotImplementedError, RuntimeError), match='jvp'):
                call()


# ---- a list far above or below the rest of the vocabulary -----------------------------------------------------------
def lists_with_a_rest(n, v, k):
    """Lists that leave 1 to 50 per cent to the rest of the vocabulary."""
    _, ids = lists_of(n, v, k, absent=False)
    left = torch.linspace(0.01, 0.5, n, device='cuda')[:, None]
    return torch.log_softmax(torch.randn(n, k, device='cuda', generator=gen(1)) * 2, -1) + torch.log1p(-left), ids


def check_far(x, t, ids, temperature):
    """The rest as an entry, in 64 bits and in logarithms, so that no distance between the list and the rest is too large:
    with w the softmax of what is off the list and P its mass, the gradient there is w (P (total + rest) - rest).

    Tolerances: the file's, and what the rest being one minus a sum in 32 bits adds: the sum is off by 2^-22 (its exponentials)
    and a few 2^-24 (its additions), 2^-21 in all, times the derivative of the loss by it."""
    from b200gdn import topk_distill_loss
    lp = torch.log_softmax(x.double() / temperature, -1)
    q = t.double().exp()
    total, given = q.sum(-1, keepdim=True), lp.gather(1, ids)
    rest = 1.0 - total
    off = lp.scatter(1, ids, -math.inf)
    log_rest, w = torch.logsumexp(off, -1, keepdim=True), torch.softmax(off, -1)
    rows = (q * (t.double() - given)).sum(-1) + (rest * (rest.log() - log_rest))[:, 0]
    size = (q * (t.double().abs() + given.abs())).sum(-1) + (rest * (rest.log().abs() + log_rest.abs() + 2.0))[:, 0]
    limit = 2.0 ** -20 + 2.0 ** -22 * size + 2.0 ** -21 * (rest.log().abs() + log_rest.abs() + 1.0)[:, 0]
    dx = (w * (log_rest.exp() * (total + rest) - rest)).scatter(1, ids, given.exp() * (total + rest) - q) / temperature
    reach = (w * (log_rest.exp() * (total + rest) + rest + 1.0)).scatter(1, ids, given.exp() * (total + rest) + q) / temperature
    options = dict(temperature=temperature, remainder='bucket')
    leaf = x.detach().requires_grad_(True)
    got = topk_distill_loss(leaf, t, ids, reduction='none', **options)
    off_by = (got.detach().double() - rows).abs()
    assert (off_by <= limit).all(), f'loss off by {off_by.tolist()}, allowed {limit.tolist()}'
    up = torch.randn(got.shape, device='cuda', generator=gen(9))
    close_grad('dlogits', torch.autograd.grad(got, leaf, up)[0], dx * up[:, None], reach * up[:, None].abs())
    total_loss = topk_distill_loss(leaf, t, ids, reduction='mean', **options)
    assert (total_loss.detach().double() - rows.mean()).abs() <= limit.mean() + 2.0 ** -22 * rows.abs().mean()
    close_grad('dlogits', torch.autograd.grad(total_loss, leaf, retain_graph=True)[0], dx / len(rows), reach / len(rows))
    close_grad('dlogits', torch.autograd.grad(0.5 * total_loss, leaf)[0], dx / (2 * len(rows)), reach / (2 * len(rows)))


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('V,k', [(70, 16), (5003, 64), (33001, 256)])
@pytest.mark.parametrize('temperature', [1.0, 0.1])
def test_distill_bucket_with_the_rest_far_away(temperature, V, k, dtype):
    """A student that puts next to nothing off the list, or on it: distances at which a mass beside the row's largest entry leaves
    what fp32 holds, as they count after the temperature; some of the rest masked."""
    gaps = [60.0, 75.0, 82.0, 84.0, 85.5, 86.0, 87.0, 88.0, 95.0, 103.0, 200.0, 700.0, 5000.0, -50.0, -86.0, -88.0, -104.0, -200.0, -5000.0]
    n = len(gaps)
    t, ids = lists_with_a_rest(n, V, k)
    x = torch.randn(n, V, device='cuda', generator=gen(2))
    x[torch.rand(n, V, device='cuda', generator=gen(3)) < 0.3] = -math.inf
    x.scatter_(1, ids, torch.randn(n, k, device='cuda', generator=gen(4)) + torch.tensor(gaps, device='cuda')[:, None])
    free = torch.ones(n, V, device='cuda').scatter_(1, ids, 0.0).argmax(-1, keepdim=True)
    x.scatter_(1, free, 0.5)     # something is left off the list
    check_far((x * temperature).to(dtype), t, ids, temperature)


@pytest.mark.parametrize('dtype', DTYPES)
def test_distill_bucket_with_one_entry_far_above_the_others(dtype):
    """Off the list one entry, and the others so far below it that they are nothing beside it, not beside the list alone."""
    n, V, k = 9, 3001, 64
    t, ids = lists_with_a_rest(n, V, k)
    x = torch.full((n, V), -200.0, device='cuda')
    free = torch.ones(n, V, device='cuda').scatter_(1, ids, 0.0).argmax(-1, keepdim=True)
    x.scatter_(1, free, -torch.tensor([80.0, 83.0, 84.0, 85.0, 86.0, 87.0, 88.0, 90.0, 120.0], device='cuda')[:, None])
    x.scatter_(1, ids, 0.0)
    check_far(x.to(dtype), t, ids, 1.0)


def test_distill_bucket_with_the_rest_at_the_lowest_values():
    """Masked with large finite numbers: a large loss, and the gradient of a uniform rest."""
    n, V, k = 4, 2000, 32
    t, ids = lists_with_a_rest(n, V, k)
    x = torch.tensor([-1e4, -1e9, -1e20, -1e30], device='cuda')[:, None].expand(n, V).contiguous()
    x.scatter_(1, ids, torch.randn(n, k, device='cuda', generator=gen(4)))
    check_far(x, t, ids, 1.0)
