"""What is done with a head's logits: log probabilities of given tokens with entropy and top alternatives, and the loss
against a teacher's top alternatives.

* ``token_logprobs`` — scoring and sampling interfaces, a teacher's pass, policy losses; differentiable.
* ``topk_distill_loss`` — a student's divergence from the entries that ``token_logprobs(..., top_k=...)`` gave of a teacher;
  the gradient of a sum or mean is formed in the same call, by a second look at the logits.

Both read logits ``[..., V]`` in bf16, fp16 or fp32 where they lie (a slice of a sequence, a padded vocabulary), hold every
sum in fp32 and run as kernels of libb200gdn.so (b200gdn_logprob_fwd/bwd, b200gdn_distill_fwd/bwd); there is no fallback path.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib
from .recorded import RecordedCall


class TokenLogprobs(NamedTuple):
    logprobs: Optional[torch.Tensor]       # [...] fp32; None without tokens
    entropy: Optional[torch.Tensor]        # [...] fp32; None where not asked for
    top_logprobs: Optional[torch.Tensor]   # [..., top_k] fp32, most probable first; None with top_k = 0
    top_ids: Optional[torch.Tensor]        # [..., top_k] int64


def _scale(who: str, temperature: float) -> float:
    if not 1e-6 <= temperature < float('inf'):
        raise ValueError(f'{who}: temperature {temperature} (at least 1e-6, finite)')
    return 1.0 / temperature


def token_logprobs(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, top_k: int = 0, temperature: float = 1.0,
                   return_entropy: bool = True) -> TokenLogprobs:
    """Log probabilities under ``softmax(logits / temperature)``.

    logits ``[..., V]``, tokens ``[...]`` (int32 or int64).  A token outside ``[0, V)``, such as the -100 of a prompt, asks
    for nothing: its log probability is 0 and has no gradient.  The ``top_k`` (up to 128) largest logits come most probable
    first, equal ones in the order of their indices.  A row whose logits are all minus infinity has log probabilities of
    minus infinity, entropy 0 and no gradient.

    Gradients of all floating results reach the logits; of ``top_logprobs`` through the entries that were chosen.
    """
    if not logits.is_cuda:
        raise _lib.B200GDNError('token_logprobs runs on a CUDA device only (no CPU path)')
    args = (logits, tokens, top_k, _scale('token_logprobs', temperature), return_entropy)
    r = _lib.host().logprob(*args)
    return TokenLogprobs(*(RecordedCall.apply(_lib.host().logprob, *args) if r is NotImplemented else r))


_REDUCTIONS = {'none': 0, 'sum': 1, 'mean': 2}


def topk_distill_loss(logits: torch.Tensor, teacher_logprobs: torch.Tensor, teacher_ids: torch.Tensor, temperature: float = 1.0,
                      remainder: str = 'renormalize', reduction: str = 'mean') -> torch.Tensor:
    """Divergence KL(q || p) of ``p = softmax(logits / temperature)`` from a teacher of whom each row has K (up to 256) entries.

    logits ``[..., V]``; teacher_logprobs ``[..., K]`` (fp32, bf16 or fp16), at the same temperature, as
    ``token_logprobs(teacher_logits, top_k=K, temperature=temperature)`` returns them; teacher_ids ``[..., K]`` (int32 or
    int64).  What the teacher leaves to the rest of the vocabulary:

    * ``remainder='renormalize'``: is dropped, q is the softmax over the entries (which takes any shift of theirs out, so
      the teacher's logits divided by the temperature serve as well);
    * ``remainder='bucket'``: is one more entry, compared with what the student leaves to the entries off the list.

    An entry with an id outside ``[0, V)`` or a log probability of minus infinity is absent.  A row without entries (a prompt) is
    left out: its loss is 0, it has no gradient and the mean does not count it.  ``reduction``: ``'mean'`` over the rows that
    count, ``'sum'`` or ``'none'`` (``[...]``).  With sum or mean and logits that require a gradient, the gradient is formed in the
    forward pass (and held until the backward pass); the backward pass only hands it on where the upstream gradient is one, else it
    forms it anew with that factor, which costs as much again: a weight or an accumulation divisor is cheaper in ``reduction='none'``,
    whose gradient is formed in the backward pass alone.
    """
    if not logits.is_cuda:
        raise _lib.B200GDNError('topk_distill_loss runs on a CUDA device only (no CPU path)')
    if remainder not in ('renormalize', 'bucket'):
        raise ValueError(f"remainder `{remainder}` is neither 'renormalize' nor 'bucket'")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction `{reduction}` is none of {', '.join(_REDUCTIONS)}")
    args = (logits, teacher_logprobs, teacher_ids, _scale('topk_distill_loss', temperature), remainder == 'bucket', _REDUCTIONS[reduction])
    loss = _lib.host().distill(*args)
    return RecordedCall.apply(_lib.host().distill, *args) if loss is NotImplemented else loss
