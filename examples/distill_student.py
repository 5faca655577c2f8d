"""A small Gated DeltaNet student learns from a teacher's top alternatives.

    python examples/distill_student.py [--steps 40]

Student and teacher are stacks of blocks ``x, stream = norm(x, stream); x = mixer(x)``: layer norm with the residual stream, then
the token mixer (projections, short convolutions, the chunked gated delta rule, the gated norm).  Each step the teacher puts out its
top log probabilities and their places (``token_logprobs``), the student its logits, and ``topk_distill_loss`` their divergence with its
gradient.  At the end the student scores tokens.  Weights and tokens are random.
"""
import argparse
import os
import sys

import torch
import torch.nn as nn

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), '..', 'flash-linear-attention_b200'))

from b200gdn import (FusedRMSNormGated, LayerNorm, ShortConvolution, chunk_gated_delta_rule, token_logprobs,  # noqa: E402
                     topk_distill_loss)


class Mixer(nn.Module):
    def __init__(self, hidden, heads, dim):
        super().__init__()
        self.heads, self.dim = heads, dim
        self.q, self.k, self.v, self.gate = (nn.Linear(hidden, heads * dim, bias=False) for _ in range(4))
        self.decay, self.beta = nn.Linear(hidden, heads, bias=False), nn.Linear(hidden, heads, bias=False)
        self.convs = nn.ModuleList(ShortConvolution(heads * dim, 4) for _ in range(3))
        self.A_log, self.dt_bias = nn.Parameter(torch.rand(heads).mul(15).add(1).log()), nn.Parameter(torch.full((heads,), -3.0))
        self.norm, self.out = FusedRMSNormGated(dim), nn.Linear(heads * dim, hidden, bias=False)

    def forward(self, x):
        split = (*x.shape[:2], self.heads, self.dim)
        q, k, v = (conv(proj(x))[0].view(split) for conv, proj in zip(self.convs, (self.q, self.k, self.v)))
        o, _ = chunk_gated_delta_rule(q, k, v, g=self.decay(x), beta=self.beta(x), use_qk_l2norm_in_kernel=True,
                                      use_gate_in_kernel=True, A_log=self.A_log, dt_bias=self.dt_bias, use_beta_sigmoid_in_kernel=True)
        return self.out(self.norm(o, self.gate(x).view(split)).flatten(-2))


class Model(nn.Module):
    def __init__(self, vocab, hidden, heads, dim, layers):
        super().__init__()
        self.embed = nn.Embedding(vocab, hidden)
        self.norms = nn.ModuleList(LayerNorm(hidden) for _ in range(layers + 1))
        self.mixers = nn.ModuleList(Mixer(hidden, heads, dim) for _ in range(layers))
        self.head = nn.Linear(hidden, vocab, bias=False)

    def forward(self, tokens):
        x, stream = self.embed(tokens), None
        for norm, mixer in zip(self.norms, self.mixers):
            x, stream = norm(x, stream, prenorm=True)
            x = mixer(x)
        return self.head(self.norms[-1](x, stream))


def main(steps=40, vocab=8000, seqs=4, length=256, top_k=32, seed=0):
    torch.manual_seed(seed)
    # computing in bf16: parameters are cast where they are used, norms and sums stay in 32 bits inside the kernels
    teacher = Model(vocab, hidden=512, heads=8, dim=64, layers=4).cuda().bfloat16()
    student = Model(vocab, hidden=256, heads=4, dim=64, layers=2).cuda().bfloat16()
    with torch.no_grad():
        teacher.head.weight.mul_(6.0)   # a teacher that prefers some tokens
    optimizer = torch.optim.AdamW(student.parameters(), lr=2e-3, weight_decay=0.0)
    tokens = torch.randint(0, vocab, (seqs, length), device='cuda')
    losses = []
    for step in range(steps):
        with torch.no_grad():
            lesson = token_logprobs(teacher(tokens), top_k=top_k, return_entropy=False)
        ids = lesson.top_ids.clone()
        ids[:, :16] = -1   # the prompt is not learned
        loss = topk_distill_loss(student(tokens), lesson.top_logprobs, ids, remainder='bucket')
        optimizer.zero_grad(set_to_none=True)
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    losses = torch.stack(losses).tolist()
    with torch.no_grad():
        scores = token_logprobs(student(tokens)[:, :-1], tokens[:, 1:], top_k=5)
    print(f'divergence from the teacher: {losses[0]:.3f} before, {losses[-1]:.3f} after {steps} steps')
    print(f'student: mean log probability {scores.logprobs.mean().item():.2f}, entropy {scores.entropy.mean().item():.2f}; '
          f'first alternatives of the last position {scores.top_ids[0, -1].tolist()}')
    return losses, scores


if __name__ == '__main__':
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument('--steps', type=int, default=40)
    main(parser.parse_args().steps)
