"""A stack of gated recurrence blocks learns to repeat its input, then writes on token by token.

    python examples/recurrent_block.py [--steps 40]

A block is ``norm -> projections -> short convolution -> gated recurrence -> gate -> projection back``, and the step between two
blocks is one pass: the norm of the block's output, its residual scale, the residual sum, the norm ahead of the next block
(``ResidualRMSNorm``).  Projections carry their activation and bias (``FusedLinear``).  While it writes, a block keeps the last inputs of its
convolution and the state of its recurrence, in place.  Weights and tokens are random.
"""
import argparse
import os
import sys

import torch
import torch.nn as nn

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), '..', 'flash-linear-attention_b200'))

from b200gdn import FusedLinear, ResidualRMSNorm, ShortConvolution, gated_recurrence, token_logprobs  # noqa: E402


class Block(nn.Module):
    def __init__(self, hidden, width):
        super().__init__()
        self.width = width
        self.into = FusedLinear(hidden, 2 * width)          # what enters the recurrence, and its forget gate
        self.gate = FusedLinear(hidden, width, activation='silu')
        self.conv = ShortConvolution(width, 4)
        self.out = FusedLinear(width, hidden, bias=False)

    def forward(self, x, cache=None):
        u, f = self.into(x).split(self.width, -1)
        conv, state = (None, None) if cache is None else cache
        u, conv = self.conv(u, cache=conv, output_final_state=cache is not None)
        # forget gates between 0.9 and 1: a channel remembers ten tokens at least
        g = 0.1 * nn.functional.logsigmoid(f)
        u = u * -torch.expm1(g)
        h, state = gated_recurrence(u, g, initial_state=state, output_final_state=cache is not None,
                                    inplace_state=state is not None and u.shape[1] == 1)
        y = self.out(h * self.gate(x))
        return y if cache is None else (y, (conv, state))


class Model(nn.Module):
    def __init__(self, vocab, hidden, width, layers):
        super().__init__()
        self.embed = nn.Embedding(vocab, hidden)
        self.first = ResidualRMSNorm(hidden)
        self.blocks = nn.ModuleList(Block(hidden, width) for _ in range(layers))
        self.between = nn.ModuleList(ResidualRMSNorm(hidden, post_norm=True, scale=0.5) for _ in range(layers))
        self.head = FusedLinear(hidden, vocab, bias=False)

    def forward(self, tokens, caches=None):
        x, stream = self.first(self.embed(tokens))
        new = []
        for i, (block, norm) in enumerate(zip(self.blocks, self.between)):
            if caches is None:
                y = block(x)
            else:
                y, cache = block(x, caches[i])
                new.append(cache)
            x, stream = norm(y, stream)
        logits = self.head(x)
        return logits if caches is None else (logits, new)

    def empty_caches(self):
        return [(None, None) for _ in self.blocks]


def main(steps=40, vocab=1024, seqs=8, length=256, write=32, seed=0):
    torch.manual_seed(seed)
    model = Model(vocab, hidden=256, width=320, layers=3).cuda().bfloat16()
    optimizer = torch.optim.AdamW(model.parameters(), lr=3e-3, weight_decay=0.0)
    tokens = torch.randint(0, vocab, (seqs, 16), device='cuda').repeat(1, length // 16)   # sixteen tokens, over and over
    losses = []
    for step in range(steps):
        loss = -token_logprobs(model(tokens[:, :-1]), tokens[:, 1:], return_entropy=False).logprobs.mean()
        optimizer.zero_grad(set_to_none=True)
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    losses = torch.stack(losses).tolist()
    with torch.no_grad():
        logits, caches = model(tokens, model.empty_caches())
        written = [logits[:, -1:].argmax(-1)]
        for _ in range(write - 1):
            logits, caches = model(written[-1], caches)
            written.append(logits.argmax(-1))
    written = torch.cat(written, 1)
    print(f'loss {losses[0]:.3f} before, {losses[-1]:.3f} after {steps} steps')
    print(f'goes on as it should in {(written == tokens[:, :write]).float().mean().item():.0%} of {written.numel()} tokens')
    return model, losses, written


if __name__ == '__main__':
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument('--steps', type=int, default=40)
    main(parser.parse_args().steps)
