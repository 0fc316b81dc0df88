"""How likely a text is: log probabilities of given tokens with the entropy and the top
alternatives of every position, from logits (``m3_token_logprobs``).

`token_logprobs` reads each logits row once and returns what evaluation, a completion API's
"logprobs" and a distillation teacher need; `train.score` runs a model in front of it, and
`distill` learns from its top alternatives.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _capi as C
from . import _tensors as T


class TokenLogprobs(NamedTuple):
    """Per row of logits, all float32 but the ids (int64); leading shape as the logits'."""

    logprob: Optional[torch.Tensor]      # log p(target), None without targets
    entropy: torch.Tensor                # of softmax(logits / temperature), in nats
    lse: torch.Tensor                    # logsumexp(logits / temperature)
    top_logprob: Optional[torch.Tensor]  # (..., top), descending, None if top == 0
    top_ids: Optional[torch.Tensor]      # (..., top)


def token_logprobs(logits: torch.Tensor, targets: Optional[torch.Tensor] = None, top: int = 0,
                   temperature: float = 1.0) -> TokenLogprobs:
    """``logits (..., V)`` bf16 or f32, ``targets (...)`` int -> `TokenLogprobs`.

    A negative target is padding: its log probability is 0; one at or past V gives NaN.  Among
    equal logits the lower id is the higher alternative.  A row whose largest logit is not
    finite (all -inf, or any +inf / NaN) has no distribution: its floats are NaN.  Views such
    as ``logits[:, :-1]`` and ``tokens[:, 1:]`` are read in place.  No gradient."""
    shape, dev = logits.shape, logits.device
    if not shape or shape[-1] < 1:
        raise ValueError(f"logits must be (..., vocab), got {tuple(shape)}")
    lead, vocab = shape[:-1], T.vocab_of(shape[-1], 1 << 30)
    T.require_here(dev, targets)
    if not 0 <= top <= min(vocab, C.M3_MAX_TOP):
        raise ValueError(f"top must be in [0, {min(vocab, C.M3_MAX_TOP)}], got {top}")
    if not temperature > 0:
        raise ValueError(f"temperature must be > 0, got {temperature}")
    dtype = T.io_dtype(logits.dtype)
    nd, f32 = len(lead), torch.float32
    outer, inner = T.row_counts(lead)
    logits, (ld_outer, ld_inner) = T.row_input(logits, nd)
    t_ptr = t_outer = t_inner = logprob = top_logprob = top_ids = None
    if targets is None:
        entropy, lse = torch.empty((2, *lead), dtype=f32, device=dev).unbind(0)
    else:
        if targets.shape != lead:
            raise ValueError(f"targets must be {tuple(lead)}, got {tuple(targets.shape)}")
        if targets.dtype != torch.int64:
            if targets.dtype != torch.int32:
                raise ValueError(f"targets must be int64 or int32, got {targets.dtype}")
            targets = targets.to(torch.int64)
        targets, (t_outer, t_inner) = T.row_input(targets, nd)
        t_ptr = targets.data_ptr()
        entropy, lse, logprob = torch.empty((3, *lead), dtype=f32, device=dev).unbind(0)
    if top:
        top_logprob = torch.empty((*lead, top), dtype=f32, device=dev)
        top_ids = torch.empty((*lead, top), dtype=torch.int64, device=dev)
    a = C.M3ScoreArgs(outer, inner, vocab, top, dtype, temperature, logits.data_ptr(), ld_outer, ld_inner, t_ptr,
                      t_outer or 0, t_inner or 0, T.ptr(logprob), entropy.data_ptr(), lse.data_ptr(),
                      T.ptr(top_logprob), T.ptr(top_ids))
    T.call(C.lib().m3_token_logprobs, a, dev)
    return TokenLogprobs(logprob, entropy, lse, top_logprob, top_ids)
