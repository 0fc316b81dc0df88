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


@torch.no_grad()
def token_logprobs(logits: torch.Tensor, targets: Optional[torch.Tensor] = None, top: int = 0,
                   temperature: float = 1.0) -> TokenLogprobs:
    """``logits (..., V)`` bf16 or f32, ``targets (...)`` int -> `TokenLogprobs`.

    A negative target is padding: its log probability is 0; one at or past V gives NaN.  Among
    equal logits the lower id is the higher alternative.  A row whose largest logit is not
    finite (all -inf, or any +inf / NaN) has no distribution: its floats are NaN.  Views such
    as ``logits[:, :-1]`` and ``tokens[:, 1:]`` are read in place.  No gradient."""
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"logits must be (..., vocab), got {tuple(logits.shape)}")
    T.require_cuda(logits, targets)
    lead, vocab = logits.shape[:-1], logits.shape[-1]
    top = int(top)
    if not 0 <= top <= min(vocab, C.M3_MAX_TOP):
        raise ValueError(f"top must be in [0, {min(vocab, C.M3_MAX_TOP)}], got {top}")
    if not temperature > 0:
        raise ValueError(f"temperature must be > 0, got {temperature}")
    if targets is not None and (targets.shape != lead or targets.device != logits.device):
        raise ValueError(f"targets must be {tuple(lead)} on {logits.device}, got {tuple(targets.shape)} on "
                         f"{targets.device}")
    if targets is not None and targets.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"targets must be int64 or int32, got {targets.dtype}")
    a = C.M3ScoreArgs()
    a.logits_dtype = T.io_dtype(logits.dtype)
    a.rows_outer, a.rows_inner = T.row_counts(lead)
    a.vocab, a.top, a.temperature = vocab, top, temperature
    nd, dev, f32 = len(lead), logits.device, torch.float32
    logits, (a.ld_outer, a.ld_inner) = T.row_input(logits, nd)
    a.logits = T.ptr(logits)
    logprob = top_logprob = top_ids = None
    if targets is not None:
        targets, (a.t_outer, a.t_inner) = T.row_input(targets.to(torch.int64), nd)
        logprob = torch.empty(lead, dtype=f32, device=dev)
        a.targets, a.logprob = T.ptr(targets), T.ptr(logprob)
    entropy, lse = torch.empty(lead, dtype=f32, device=dev), torch.empty(lead, dtype=f32, device=dev)
    a.entropy, a.lse = T.ptr(entropy), T.ptr(lse)
    if top:
        top_logprob = torch.empty(*lead, top, dtype=f32, device=dev)
        top_ids = torch.empty(*lead, top, dtype=torch.int64, device=dev)
        a.top_logprob, a.top_ids = T.ptr(top_logprob), T.ptr(top_ids)
    T.call(C.lib().m3_token_logprobs, a, dev)
    return TokenLogprobs(logprob, entropy, lse, top_logprob, top_ids)
