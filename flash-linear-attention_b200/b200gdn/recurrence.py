"""The elementwise gated recurrence: the token mixer of recurrent blocks that stand between those of the delta rule, behind the same
short convolution.

``gated_recurrence`` — ``h_t = exp(g_t) h_{t-1} + x_t`` along each sequence, differentiable, with the states that a serving loop
carries from call to call.  It runs as a kernel of libb200gdn.so (b200gdn_gated_recurrence_fwd/bwd); there is no fallback path.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from .index import tables_for
from .recorded import RecordedCall, recorded


def _native(x, g, initial_state, output_final_state, inplace_state, cu_seqlens, cu_seqlens_cpu):
    if cu_seqlens is None:
        return _lib.host().gated_recurrence(x, g, initial_state, output_final_state, inplace_state, None, 0)
    tables = tables_for(x.shape[0], x.shape[1], cu_seqlens, cu_seqlens_cpu, x.device)
    return _lib.host().gated_recurrence(x, g, initial_state, output_final_state, inplace_state, tables.native(), tables.longest)


def gated_recurrence(
    x: torch.Tensor,
    g: torch.Tensor,
    initial_state: Optional[torch.Tensor] = None,
    output_final_state: bool = False,
    cu_seqlens: Optional[torch.Tensor] = None,
    cu_seqlens_cpu: Optional[torch.Tensor] = None,
    inplace_state: bool = False,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``h_t = exp(g_t) h_{t-1} + x_t`` for every channel of every sequence; returns ``(h, final_state)``.

    x, g ``[B,T,D]`` in bf16, fp16 or fp32 (``B == 1`` with ``cu_seqlens [N+1]``, whose sequences lie one behind the other); slices of a
    wider projection are read where they lie.  g is the logarithm of a decay, as the mixers' gates are: 0 keeps, minus infinity forgets.
    (Above 0 a state grows; products of ``exp(g)`` over up to 2048 neighbouring tokens must stay below 2^127 then.)  A decay below 2^-126.5 counts
    as zero; while decays are not zero an infinite state stays infinite.  A g that has neither the type of x nor fp32 is cast to fp32.

    ``initial_state [N,D]`` (zeros where absent) and ``final_state [N,D]`` in fp32; everything in between is held in fp32 too, and
    gradients, which reach x, g and initial_state from both results, are formed from states that were not rounded.  A sequence without
    tokens hands its state on.  Rows that no sequence covers are zero in h and in the gradients.  ``inplace_state=True`` (without
    gradients, with ``output_final_state``) writes the final state over ``initial_state``, which has to be fp32 and contiguous.
    """
    if not x.is_cuda:
        raise _lib.B200GDNError('gated_recurrence runs on a CUDA device only (no CPU path)')
    if x.dim() != 3:
        raise _lib.B200GDNError(f'gated_recurrence: x is [batch, tokens, channels], got {tuple(x.shape)}')
    if cu_seqlens is not None and x.shape[0] != 1:
        raise ValueError(f"The batch size is expected to be 1 rather than {x.shape[0]} when using `cu_seqlens`.")
    if inplace_state and not output_final_state:
        raise ValueError('`inplace_state` hands the final state back: it needs `output_final_state`')
    args = (x, g, initial_state, output_final_state, inplace_state, cu_seqlens, cu_seqlens_cpu)
    return RecordedCall.apply(_native, *args) if recorded(x) else _native(*args)
