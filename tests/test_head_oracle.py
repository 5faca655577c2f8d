"""The 64-bit restatements in oracle/head_oracle.py against differences and against torch's own derivatives, on the CPU."""
import math

import pytest
import torch

from oracle import head_oracle as H

STEP = 1e-6
# central differences of a smooth function in 64 bits: truncation STEP^2 (about 1e-12 x third derivative), rounding 1e-16 / STEP x value
TOL = 1e-8


def _differences(f, x):
    g = torch.zeros_like(x)
    flat, out = x.view(-1), g.view(-1)
    for i in range(flat.numel()):
        keep = flat[i].item()
        flat[i] = keep + STEP
        up = f(x)
        flat[i] = keep - STEP
        out[i] = (up - f(x)) / (2 * STEP)
        flat[i] = keep
    return g


def test_layer_norm_gradient_is_that_of_differences():
    torch.manual_seed(0)
    x, w, b, dy, dz = torch.randn(3, 7).double(), torch.randn(7).double(), torch.randn(7).double(), torch.randn(3, 7).double(), torch.randn(3, 7).double()
    got = H.layer_norm(x, w, b, None, 1e-5, dy, dz)

    def f(x, w, b):
        return ((H.layer_norm(x, w, b, None, 1e-5)['y'] * dy).sum() + (x * dz).sum()).item()
    assert (got['dx'] - _differences(lambda v: f(v, w, b), x)).abs().max() < 10 * TOL
    assert (got['dweight'] - _differences(lambda v: f(x, v, b), w)).abs().max() < 10 * TOL
    assert (got['dbias'] - _differences(lambda v: f(x, w, v), b)).abs().max() < 10 * TOL


@pytest.mark.parametrize('temperature', [1.0, 0.7])
def test_logprobs_gradient_is_that_of_differences(temperature):
    torch.manual_seed(1)
    x, tokens = torch.randn(4, 9).double() * 2, torch.tensor([3, -100, 8, 9])
    x[2, 4] = -math.inf
    dlp, dh, dtop = torch.randn(4).double(), torch.randn(4).double(), torch.randn(4, 3).double()

    def f(v):
        o = H.logprobs(v, tokens, 3, temperature)
        return ((o['logprobs'] * dlp).sum() + (o['entropy'] * dh).sum() + (o['top_logprobs'] * dtop).sum()).item()
    got, want = H.logprobs(x, tokens, 3, temperature, dlp, dh, dtop)['dx'], _differences(f, x)
    want[2, 4] = 0.0   # of minus infinity there are no differences
    assert (got - want).abs().max() < 10 * TOL


@pytest.mark.parametrize('bucket', [False, True])
def test_distill_gradient_is_that_of_differences(bucket):
    torch.manual_seed(2)
    x = torch.randn(5, 11).double() * 2
    ids = torch.tensor([[3, 1, 7], [0, -1, 2], [4, 4, 10], [-1, -1, -1], [5, 11, 6]])
    teacher = torch.log_softmax(torch.randn(5, 4).double(), -1)[:, :3].contiguous()
    teacher[4, 2] = -math.inf
    got = H.distill(x, teacher, ids, 1.7, bucket)
    assert got['counted'].tolist() == [True, True, True, False, True]
    want = _differences(lambda v: H.distill(v, teacher, ids, 1.7, bucket)['rows'].sum().item(), x)
    assert (got['dx'] - want).abs().max() < 10 * TOL
    assert got['rows'][3] == 0 and (got['rows'][[0, 1, 2, 4]] > 0).all()


def test_against_torch():
    """log_softmax, its derivative, kl_div and layer_norm of torch in 64 bits."""
    torch.manual_seed(3)
    x, tokens = torch.randn(6, 40).double().requires_grad_(True), torch.randint(0, 40, (6,))
    lp = torch.log_softmax(x / 1.3, -1)
    ent = torch.distributions.Categorical(logits=x / 1.3).entropy()
    got = H.logprobs(x.detach(), tokens, 5, 1.3, torch.ones(6), torch.full((6,), 0.5))
    assert torch.allclose(got['logprobs'], lp.gather(1, tokens[:, None])[:, 0], atol=1e-13) and torch.allclose(got['entropy'], ent, atol=1e-13)
    dx, = torch.autograd.grad(lp.gather(1, tokens[:, None]).sum() + 0.5 * ent.sum(), x)
    assert torch.allclose(got['dx'], dx, atol=1e-13)
    # a teacher's whole distribution as a list: the ordinary divergence
    t = torch.log_softmax(torch.randn(6, 40).double(), -1)
    ids = torch.stack([torch.randperm(40) for _ in range(6)])
    want = torch.nn.functional.kl_div(torch.log_softmax(x, -1), t, log_target=True, reduction='sum')
    dx, = torch.autograd.grad(want, x)
    for bucket in (False, True):
        d = H.distill(x.detach(), t.gather(1, ids), ids, 1.0, bucket)
        assert torch.allclose(d['rows'].sum(), want.detach(), atol=1e-12)
        assert torch.allclose(d['dx'], dx, atol=1e-12)
    y = torch.nn.functional.layer_norm(x, (40,), eps=1e-5)
    assert torch.allclose(H.layer_norm(x.detach(), None, None, None, 1e-5)['y'], y.detach(), atol=1e-12)
