"""Distillation from a teacher's top logits, with hard labels mixed in (``m3_distill``).

Per row x of student logits, with p the softmax of the teacher's k logits over T:

    loss = w [ (1 - hard_weight) T^2 KL(p || softmax(x / T)) + hard_weight CE(x, label) ]

`distill_loss` is an autograd function; `distill_loss_and_grad` gives the loss and the gradient
with respect to the logits together, from one read of them (`train.make_distill_step`).  The
teacher's lists are `scoring.token_logprobs`' ``top_ids`` and ``top_logprob``.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _capi as C
from . import _tensors as T

_REDUCE = {"none": C.M3_REDUCE_NONE, "sum": C.M3_REDUCE_SUM, "mean": C.M3_REDUCE_MEAN}


def _side(name, t, shape, dtype, others):
    """A side input as the kernel reads it: dense, int64 or f32."""
    if t.shape != shape:
        raise ValueError(f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")
    if t.dtype != dtype:
        if not others(t.dtype):
            raise ValueError(f"{name} must be {'integers' if dtype == torch.int64 else 'floating point'}, got {t.dtype}")
        t = t.detach().to(dtype)
    return t if t.is_contiguous() else t.detach().contiguous()


def _is_int(dt):
    return dt == torch.int32


def _is_float(dt):
    return dt.is_floating_point


def _check(logits, ids, teacher, labels, weights, temperature, hard_weight, reduction):
    """Argument checks; returns the side inputs as the kernel reads them (dense int64 / f32)."""
    shape = logits.shape
    if not shape or shape[-1] < 1:
        raise ValueError(f"logits must be (..., vocab), got {tuple(shape)}")
    T.vocab_of(shape[-1], 1 << 30)
    T.require_here(logits.device, ids, teacher, labels, weights)
    lead = shape[:-1]
    k = ids.shape[-1] if ids.dim() else 0
    if not 1 <= k <= C.M3_MAX_TOP:
        raise ValueError(f"teacher_ids must be {tuple(lead)} + (k,), 1 <= k <= {C.M3_MAX_TOP}, got {tuple(ids.shape)}")
    if not temperature > 0 or not 0 <= hard_weight <= 1:
        raise ValueError("need temperature > 0 and 0 <= hard_weight <= 1")
    if reduction not in _REDUCE:
        raise ValueError(f"reduction must be one of {sorted(_REDUCE)}, got {reduction!r}")
    if (labels is not None) != (hard_weight > 0):
        raise ValueError("labels go with hard_weight > 0")
    entries = (*lead, k)
    ids = _side("teacher_ids", ids, entries, torch.int64, _is_int)
    teacher = _side("teacher_logits", teacher, entries, torch.float32, _is_float)
    if labels is not None:
        labels = _side("labels", labels, lead, torch.int64, _is_int)
    if weights is not None:
        weights = _side("weights", weights, lead, torch.float32, _is_float)
    return ids, teacher, labels, weights


def _run(logits, ids, teacher, labels, weights, temperature, hard_weight, reduction, grad=None, upstream=None,
         grad_scale=1.0, weight_sum=None, want_loss=True, ready=0):
    """One m3_distill call on checked inputs: the reduced loss, or the rows' losses (None unless
    wanted).  ``weight_sum``: one float that a mean with weights leaves their sum in."""
    lead, dev = logits.shape[:-1], logits.device
    nd = len(lead)
    outer, inner = T.row_counts(lead)
    logits, (ld_outer, ld_inner) = T.row_input(logits, nd)
    g_outer, g_inner = (0, 0) if grad is None else T.rows2(grad, nd)
    result = rows_at = loss_at = None
    sum_at = T.ptr(weight_sum)
    if want_loss and reduction == "none":
        result = torch.empty(lead, dtype=torch.float32, device=dev)
        rows_at = result.data_ptr()
    elif want_loss:
        result = torch.empty((), dtype=torch.float32, device=dev)
        work = torch.empty(1 + outer * inner, dtype=torch.float32, device=dev)  # sum of weights, rows' losses
        loss_at, rows_at = result.data_ptr(), work.data_ptr() + 4
        sum_at = sum_at or work.data_ptr()
    stride = 0 if upstream is None or upstream.dim() == 0 or upstream.numel() == 1 else 1
    a = C.M3DistillArgs(outer, inner, logits.shape[-1], ids.shape[-1], T.io_dtype(logits.dtype), _REDUCE[reduction],
                        temperature, hard_weight, grad_scale, logits.data_ptr(), ld_outer, ld_inner, ids.data_ptr(),
                        teacher.data_ptr(), T.ptr(labels), T.ptr(weights), T.ptr(upstream), stride, rows_at, loss_at,
                        sum_at, T.ptr(grad), g_outer, g_inner, ready, 0)
    T.call(C.lib().m3_distill, a, dev)
    return result


class _DistillFn(torch.autograd.Function):
    """A reduced loss comes with its gradient from one read of the logits: the backward, whose
    upstream gradient is 1 in a plain ``loss.backward()``, then only looks at that and returns it; with
    another upstream (or a second backward) it reads the logits again.  The rows' losses have one upstream
    each, so theirs is always written in the backward."""

    @staticmethod
    def forward(ctx, logits, ids, teacher, labels, weights, temperature, hard_weight, reduction):
        ctx.save_for_backward(logits, ids, teacher, labels, weights)
        ctx.opts = (temperature, hard_weight, reduction)
        ctx.grad = ctx.weight_sum = None
        if reduction != "none":
            ctx.grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
            if weights is not None:
                ctx.weight_sum = torch.empty(1, dtype=torch.float32, device=logits.device)
        return _run(logits, ids, teacher, labels, weights, *ctx.opts, grad=ctx.grad, weight_sum=ctx.weight_sum)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss):
        saved = ctx.saved_tensors
        logits, weights = saved[0], saved[4]
        grad, ctx.grad = ctx.grad, None  # handed out once: its next owner may write to it
        ready = 0 if grad is None else C.M3_READY_GRAD
        if grad is None:
            grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        total = ctx.weight_sum
        if total is not None:
            ready |= C.M3_READY_WEIGHTS
        _run(*saved, *ctx.opts, grad=grad, upstream=dloss.float().contiguous(), weight_sum=total, want_loss=False,
             ready=ready)
        return (grad,) + (None,) * 7


def distill_loss(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor, *,
                 temperature: float = 1.0, labels: Optional[torch.Tensor] = None, hard_weight: float = 0.0,
                 weights: Optional[torch.Tensor] = None, reduction: str = "mean") -> torch.Tensor:
    """The loss of ``logits (..., V)`` (bf16 or f32) against ``teacher_ids`` / ``teacher_logits``
    ``(..., k)``, k <= 128; differentiable in ``logits`` alone, once and in reverse mode.

    A negative id is an absent entry, a negative label an absent label; the teacher's logits
    may be shifted by any constant (log probabilities do).  ``weights (...)`` weigh the rows; a
    row of weight 0, or with neither entries nor label, contributes exactly 0 to the loss and
    the gradient whatever its logits are.  An id or label at or past V makes its row NaN.
    ``reduction``: "mean" over the weights' sum (or the row count), "sum", or "none" for the
    rows' losses.  A mean over weights that are all 0 is 0 (a rank's shard of padding).
    ``temperature``: 1e-30 to 1e18; the loss holds T^2 times the rounding of fp32 logarithms (some
    1e-7), the gradient T times that of fp32 probabilities.

    With gradients enabled a "mean" or "sum" forms the gradient together with the loss, in memory of
    the logits' size that the backward hands on; a backward whose upstream gradient is not 1 (a
    scaled loss) reads the logits again, where `distill_loss_and_grad`'s ``grad_scale`` does not."""
    T.no_tangent("distill_loss", logits)
    side = _check(logits, teacher_ids, teacher_logits, labels, weights, temperature, hard_weight, reduction)
    if torch.is_grad_enabled() and logits.requires_grad:
        return _DistillFn.apply(logits, *side, float(temperature), float(hard_weight), reduction)
    return _run(logits, *side, temperature, hard_weight, reduction)


def distill_loss_and_grad(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor, *,
                          temperature: float = 1.0, labels: Optional[torch.Tensor] = None, hard_weight: float = 0.0,
                          weights: Optional[torch.Tensor] = None, reduction: str = "mean", grad_scale: float = 1.0,
                          out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """`distill_loss` ("mean" or "sum") and ``grad_scale`` times its gradient with respect to the
    logits, in the logits' dtype, from one read of them.  ``out`` takes the gradient; it may be
    ``logits`` itself, which are then overwritten: as after any in-place operation, a backward
    that saved them raises."""
    if reduction == "none":
        raise ValueError("reduction must be 'mean' or 'sum'")
    side = _check(logits, teacher_ids, teacher_logits, labels, weights, temperature, hard_weight, reduction)
    nd = logits.dim() - 1
    given = out is not None
    if not given:
        out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    elif out.requires_grad and out.is_leaf and torch.is_grad_enabled():
        raise ValueError("out must not be a leaf that requires grad")
    elif out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device:
        raise ValueError(f"out must be {tuple(logits.shape)} {logits.dtype} on {logits.device}")
    elif not _writable_rows(out, nd):
        raise ValueError("out must have a contiguous vocabulary axis and rows that do not overlap")
    elif not (out.data_ptr() == logits.data_ptr() and out.stride() == logits.stride()) and not T.apart(out, logits):
        raise ValueError("out must be the logits themselves or share no memory with them")
    loss = _run(logits, *side, temperature, hard_weight, reduction, grad=out, grad_scale=grad_scale)
    if given:
        T.written(out)
    return loss, out


def _writable_rows(t, nd) -> bool:
    if t.numel() == 0:
        return True
    st = T.rows2(t, nd)
    if st is None or (t.shape[-1] > 1 and t.stride(-1) != 1):
        return False
    outer, inner = T.row_counts(t.shape[:-1])
    span = t.shape[-1]
    for count, stride in sorted(((inner, st[1]), (outer, st[0])), key=lambda cs: cs[1]):
        if count > 1:
            if stride < span:
                return False
            span = stride * (count - 1) + span
    return True
