"""The operators of a gated recurrence block in processes and runs of their own."""
import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), '..'))

FIRST_CALL = '''
import sys
sys.path.insert(0, 'flash-linear-attention_b200')
import torch, b200gdn
x = torch.randn(2, 300, 64, device='cuda', dtype=torch.bfloat16)
{make}
loss = y.sum()
loss.backward()
torch.cuda.synchronize()
print('done', torch.isfinite(leaf.grad).all().item())
'''


@pytest.mark.parametrize('make', ['leaf = -x.abs(); leaf.requires_grad_(True); y, _ = b200gdn.gated_recurrence(x, leaf)',
                                  'leaf = torch.randn(72, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True); y = b200gdn.fused_linear(x, leaf)',
                                  'leaf = x.clone().requires_grad_(True); y, _ = b200gdn.residual_rms_norm(leaf, residual=x)'])
def test_the_first_backward_pass_of_a_process(make):
    """It runs on a thread that has made no CUDA call yet."""
    out = subprocess.run([sys.executable, '-c', FIRST_CALL.format(make=make)], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and 'done True' in out.stdout, out.stderr[-2000:]


def plain_block(block, x, h0=None):
    """The block of examples/recurrent_block.py in 64 bits and elementary operations; parameters by name in `block`."""
    z = x @ block['into.weight'].t() + block['into.bias']
    W = block['conv.weight'].shape[0]
    u, f = z[..., :W], z[..., W:]
    taps = block['conv.weight'].view(W, -1)
    padded = torch.cat([u.new_zeros(u.shape[0], taps.shape[1] - 1, W), u], 1)
    u = sum(padded[:, i:i + u.shape[1]] * taps[:, i] for i in range(taps.shape[1]))
    u = u * torch.sigmoid(u)
    g = 0.1 * torch.nn.functional.logsigmoid(f)
    u = u * -torch.expm1(g)
    h, rows = u.new_zeros(u.shape[0], W), []
    for t in range(u.shape[1]):
        h = torch.exp(g[:, t]) * h + u[:, t]
        rows.append(h)
    gate = x @ block['gate.weight'].t() + block['gate.bias']
    return (torch.stack(rows, 1) * (gate * torch.sigmoid(gate))) @ block['out.weight'].t()


def test_a_block_with_the_steps_around_it():
    """Norm, projections, convolution, recurrence, gate, projection, and the step to the next block, with the gradients of all parameters, in
    fp16 against 64 bits.

    Ten times on the way to the result a tensor is rounded to fp16, half a step (2^-11) of its own size at most, and what follows carries
    that on with a factor around one (norms keep relative errors, the gates' slopes are below 1.1, decays below one): 10 x 2^-11 = 0.5 %
    of the norm of the whole.  A gradient passes each rounding's place twice, there and back: 1 %."""
    sys.path.insert(0, os.path.join(ROOT, 'examples'))
    try:
        from recurrent_block import Block
    finally:
        sys.path.pop(0)
    from b200gdn import ResidualRMSNorm
    torch.manual_seed(0)
    HF, hidden, width = torch.float16, 96, 136
    block = Block(hidden, width).cuda().to(HF)
    first, after = ResidualRMSNorm(hidden).cuda().to(HF), ResidualRMSNorm(hidden, post_norm=True, scale=0.5).cuda().to(HF)
    x = torch.randn(2, 75, hidden, device='cuda').to(HF).requires_grad_(True)
    n, stream = first(x)
    out, z = after(block(n), stream)
    ups = [torch.randn_like(out), torch.randn_like(out)]
    named = [('x', x)] + [(f'{m}.{k}', p) for m, mod in (('block', block), ('first', first), ('after', after)) for k, p in mod.named_parameters()]
    got = torch.autograd.grad([out, z], [p for _, p in named], ups)
    d = {k: p.detach().double().requires_grad_(True) for k, p in named}

    def rms(v):
        return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-6)
    stream = d['x']
    y = plain_block({k[6:]: v for k, v in d.items() if k.startswith('block.')}, rms(stream) * d['first.weight'])
    z64 = stream + d['after.scale'] * rms(y) * d['after.post_weight']
    out64 = rms(z64) * d['after.weight']
    want = torch.autograd.grad([out64, z64], list(d.values()), [u.double() for u in ups])
    for name, a, b in [('out', out, out64), ('z', z, z64)]:
        assert (a.detach().double() - b.detach()).norm() <= 5e-3 * b.detach().norm(), name
    for (name, _), a, b in zip(named, got, want):
        assert (a.double() - b).norm() <= 1e-2 * b.norm(), (name, ((a.double() - b).norm() / b.norm()).item())


def test_the_example_runs_and_writes_as_it_reads():
    """Its loss is a number, every parameter has a gradient, and token by token the model gives what it gives for the sequence at once: to the
    rounding of bf16 (2^-8 of the largest logit for each of some ten roundings a block)."""
    sys.path.insert(0, os.path.join(ROOT, 'examples'))
    try:
        import recurrent_block
    finally:
        sys.path.pop(0)
    model, losses, written = recurrent_block.main(steps=3, vocab=96, seqs=3, length=64, write=4)
    assert all(l == l for l in losses) and written.shape == (3, 4)
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in model.parameters())
    tokens = torch.randint(0, 96, (3, 40), device='cuda')
    with torch.no_grad():
        whole = model(tokens).float()
        first, caches = model(tokens[:, :20], model.empty_caches())
        parts = [first]
        for t in range(20, 40):
            logits, caches = model(tokens[:, t:t + 1], caches)
            parts.append(logits)
    parts = torch.cat(parts, 1).float()
    assert (parts - whole).abs().max() <= 40 * 2.0 ** -8 * whole.abs().max()


def test_two_captured_graphs_of_one_model_replay_in_turn():
    """Workspaces belong to their calls: two graphs of the same operators, replayed one after the other and at the same time on two streams."""
    from b200gdn import fused_linear, gated_recurrence, residual_rms_norm
    g = torch.Generator('cuda').manual_seed(0)
    data = [[torch.randn(2, 300, 72, device='cuda', generator=g).bfloat16() for _ in range(2)] for _ in range(2)]
    w = torch.randn(72, 72, device='cuda', generator=g).bfloat16()

    def run(x, f):
        y = fused_linear(x, w, activation='silu')
        h, s = gated_recurrence(y, -f.abs(), output_final_state=True)
        out, z = residual_rms_norm(h, residual=x, post_norm=True)
        return out, z, s
    want = [[t.clone() for t in run(*d)] for d in data]
    graphs, outs = [], []
    for d in data:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run(*d))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for s, graph in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graph.replay()
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        for o, r in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(o, r))
