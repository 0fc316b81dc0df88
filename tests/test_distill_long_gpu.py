"""Distillation of long rows by one CTA each (more rows than half the SMs, so that no row is shared by a
cluster): rows read again from L2, wider CTAs, repeated ids past the search bits, any alignment, in place.

Tolerances: an element is factor * 2^d with |d| < 40 (6e-6 relative, as in test_distill_gpu); 2e-5 relative,
and 2^-8 for bf16's rounding.  At a teacher's id or a label the target is subtracted, which adds 2e-6 of the
row's factor; nowhere else, so that an element left out or written twice shows at any size."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _inputs(rows, vocab, k, dtype, hard, repeated):
    g = torch.Generator(device="cuda").manual_seed(vocab + k)
    rand = lambda *s: torch.rand(*s, generator=g, device="cuda")
    x = (torch.randn(rows, vocab, generator=g, device="cuda") * 2).to(dtype)
    ids = (torch.randint(0, vocab, (rows, 1), generator=g, device="cuda") +
           torch.arange(k, device="cuda") * (vocab // k)) % vocab
    ids[:, k // 2][rand(rows) < 0.3] = -1
    ids[0, :2] = torch.tensor([0, vocab - 1], device="cuda")  # the row's ends
    if repeated:
        ids[1::3, 1::2] = ids[1::3, :1]
        ids[2] = vocab // 2
    teacher = torch.randn(rows, k, generator=g, device="cuda") * 2
    labels = torch.where(rand(rows) < 0.5, ids[:, 0], 3) if hard else None
    weights = (rand(rows) < 0.9).float()
    weights[:3] = 1.0
    return x, ids, teacher, labels, weights


def _formulas(x, ids, teacher, labels, weights, T, hard):
    """Loss, gradient, and the elements where a target is subtracted, in 64 bits."""
    there = ids >= 0
    at = ids.clamp_min(0)
    p = torch.nan_to_num(torch.softmax(torch.where(there, teacher.double() / T, -math.inf), 1))
    logq = torch.log_softmax(x.double() / T, 1)
    terms = p * (torch.log(p) - logq.gather(1, at))
    rows = (1 - hard) * T * T * torch.where(p > 0, terms, 0.0).sum(1)
    grad = (1 - hard) * T * there.any(1).double()[:, None] * torch.exp(logq)
    grad.scatter_add_(1, at, -(1 - hard) * T * p)
    target = torch.zeros(x.shape, dtype=torch.int32, device="cuda").scatter_add_(1, at, there.int())
    if hard:
        on, lab = (labels >= 0).double(), labels.clamp_min(0)[:, None]
        logq = torch.log_softmax(x.double(), 1)
        rows = rows - hard * on * logq.gather(1, lab)[:, 0]
        grad += hard * on[:, None] * torch.exp(logq)
        grad.scatter_add_(1, lab, -hard * on[:, None])
        target.scatter_add_(1, lab, on.int()[:, None])
    w = weights.double()
    return float((rows * w).sum() / w.sum()), grad * (w / w.sum())[:, None], target > 0


def _check(got, want, target, weights, T, dtype):
    rtol = 2e-5 + (2.0 ** -8 if dtype == BF else 0.0)
    coef = (weights.double() / weights.double().sum() * max(1.0, T))[:, None]
    bound = rtol * want.abs() + torch.where(target, 2e-6 * coef, 0.0)
    assert ((got.double() - want).abs() <= bound).all()  # a NaN is not within it
    assert not got[weights == 0].any()


CASES = [
    (100, 128256, 64, BF, 0.0, False),   # three tiles: the last from L2
    (100, 128256, 20, BF, 0.4, True),
    (100, 50257, 32, F32, 0.3, False),
    (100, 100003, 16, F32, 0.0, True),   # wider CTAs
    (80, 140001, 24, BF, 0.0, True),     # more elements than search bits
    (80, 140001, 24, F32, 0.3, True),
    (80, 262147, 128, BF, 0.0, True),
    (400, 50257, 8, BF, 0.0, False),
]


@pytest.mark.parametrize("rows,vocab,k,dtype,hard,repeated", CASES)
def test_long_rows_by_one_cta(rows, vocab, k, dtype, hard, repeated):
    from mamba3_b200 import distill as D

    x, ids, teacher, labels, weights = _inputs(rows, vocab, k, dtype, hard, repeated)
    T = 1.7
    want, grad, target = _formulas(x, ids, teacher, labels, weights, T, hard)
    tol = (1 + T * T) * (8e-6 + 1e-6 * float(x.float().abs().max())) + 2e-6 * abs(want)
    args = dict(temperature=T, labels=labels, hard_weight=hard, weights=weights)
    out = torch.full_like(x, math.nan)
    loss, dx = D.distill_loss_and_grad(x, ids, teacher, out=out, **args)
    assert abs(float(loss) - want) <= tol
    _check(dx, grad, target, weights, T, dtype)
    with torch.no_grad():
        assert abs(float(D.distill_loss(x, ids, teacher, **args)) - want) <= tol
    # rows at an odd offset and pitch, the gradient beside them at another
    buf = torch.full((rows, vocab + 13), math.nan, dtype=dtype, device="cuda")
    view = buf[:, 5:5 + vocab]
    view.copy_(x)
    side = torch.full((rows, vocab + 6), 7.0, dtype=dtype, device="cuda")
    loss, dx = D.distill_loss_and_grad(view, ids, teacher, out=side[:, 2:2 + vocab], **args)
    assert abs(float(loss) - want) <= tol
    _check(dx, grad, target, weights, T, dtype)
    assert (side[:, :2] == 7).all() and (side[:, 2 + vocab:] == 7).all()
    # in place, at that offset and aligned
    loss, dx = D.distill_loss_and_grad(view, ids, teacher, out=view, **args)
    assert abs(float(loss) - want) <= tol and torch.isnan(buf[:, :5]).all() and torch.isnan(buf[:, 5 + vocab:]).all()
    _check(dx, grad, target, weights, T, dtype)
    leaf = x.clone().requires_grad_(True)
    D.distill_loss(leaf, ids, teacher, **args).backward()
    _check(leaf.grad, grad, target, weights, T, dtype)
    loss, dx = D.distill_loss_and_grad(x, ids, teacher, out=x, **args)
    assert dx is x and abs(float(loss) - want) <= tol
    _check(x, grad, target, weights, T, dtype)
