"""`distill.distill_loss` and `distill_loss_and_grad` against the 64-bit formulas, their autograd
and differences.

Tolerances: fp32 arithmetic; a softmax value is off by 2^-22 + |d| 2^-23 relative with
|d| < 40 here (6e-6), a log probability by 4e-6 + 3e-7 of the logits' size, and T^2 multiplies
the loss.  An fp32 gradient is therefore within 2e-5 relative plus 2e-6 of its coefficient
(where the teacher's share cancels), a bf16 one within its rounding (2^-8 relative) besides."""

import math

import pytest
import torch

from tests import vocab_ref as R

CUDA = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _case(rows, vocab, k, dtype, seed, hard=0.0, weighted=False, lead=None):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, vocab, generator=g) * 2).to(dtype)
    ids = torch.stack([torch.randperm(vocab, generator=g)[:k] if k <= vocab else
                       torch.randint(0, vocab, (k,), generator=g) for _ in range(rows)])
    teacher = torch.randn(rows, k, generator=g).sort(dim=1, descending=True).values * 2
    ids[torch.rand(rows, k, generator=g) < 0.15] = -1
    labels = torch.randint(0, vocab, (rows,), generator=g) if hard > 0 else None
    if labels is not None:
        some = torch.rand(rows, generator=g)
        labels = torch.where(some < 0.4, ids[:, 0], labels)  # the label among the teacher's ids
        labels[some > 0.8] = -100
    weights = (torch.rand(rows, generator=g) * (torch.rand(rows, generator=g) < 0.8)) if weighted else None
    if weighted:
        weights[0] = 1.0
    return x, ids, teacher, labels, weights


def _cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


def _want(x, ids, teacher, labels, weights, temperature, hard, reduction, upstream=None):
    xd = x.double().clone().requires_grad_(True)
    rows = R.distill_rows(xd, ids, teacher, labels, weights, temperature, hard)
    loss = R.reduce(rows, weights, reduction)
    grad = torch.autograd.grad(loss, xd, upstream)[0] if loss.requires_grad else torch.zeros_like(xd)
    return loss.detach(), grad


def _check_grad(got, want, coef, dtype, what):
    """`coef`: the largest factor in front of a softmax, per row (R, 1) or one number."""
    got = got.double().cpu()
    assert got.shape == want.shape
    rtol = 2e-5 + (2.0 ** -8 if dtype == BF else 0.0)
    err = (got - want).abs() - rtol * want.abs() - 2e-6 * coef
    assert float(err.max()) <= 0, (what, float(err.max()))
    zero = (want == 0).all(1)  # rows that contribute nothing: exactly nothing
    assert torch.equal(got[zero], torch.zeros_like(got[zero]))


def _loss_tol(temperature, x, loss):
    return (1 + temperature ** 2) * (8e-6 + 1e-6 * float(x.float().abs().max())) + 2e-6 * abs(loss)


def _check(x, ids, teacher, labels, weights, temperature, hard):
    from mamba3_b200 import distill as D

    dtype = x.dtype
    cx, cids, ct, cl, cw = _cuda(x, ids, teacher, labels, weights)
    args = dict(temperature=temperature, labels=cl, hard_weight=hard, weights=cw)
    rows, _ = _want(x, ids, teacher, labels, weights, temperature, hard, "none", torch.ones(x.shape[0]).double())
    got = D.distill_loss(cx, cids, ct, reduction="none", **args)
    for r in range(x.shape[0]):
        assert abs(float(got[r]) - float(rows[r])) <= _loss_tol(temperature, x, float(rows[r])), r
    w = torch.ones(x.shape[0]).double() if weights is None else weights.double()
    for reduction in ("mean", "sum"):
        want, grad = _want(x, ids, teacher, labels, weights, temperature, hard, reduction)
        div = float(w.sum()) if reduction == "mean" else 1.0
        coef = (w / div * max(1.0, temperature))[:, None]
        tol = _loss_tol(temperature, x, float(want)) * (1.0 if reduction == "mean" else float(w.sum()))
        loss, dx = D.distill_loss_and_grad(cx, cids, ct, reduction=reduction, **args)
        assert abs(float(loss) - float(want)) <= tol
        _check_grad(dx, grad, coef, dtype, reduction)
        leaf = cx.clone().requires_grad_(True)
        loss2 = D.distill_loss(leaf, cids, ct, reduction=reduction, **args)
        (loss2 * 3.0).backward()
        assert abs(float(loss2) - float(want)) <= tol
        _check_grad(leaf.grad, 3.0 * grad, 3.0 * coef, dtype, reduction + " autograd")
    # every row with a gradient of its own
    up = torch.randn(x.shape[0], generator=torch.Generator().manual_seed(8))
    _, grad = _want(x, ids, teacher, labels, weights, temperature, hard, "none", up.double())
    leaf = cx.clone().requires_grad_(True)
    D.distill_loss(leaf, cids, ct, reduction="none", **args).backward(up.cuda())
    _check_grad(leaf.grad, grad, (w * up.double().abs() * max(1.0, temperature))[:, None], dtype, "rows")


SIZES = [1, 2, 9, 32, 255, 256, 257, 513, 1000, 1025, 2049, 4097, 8193, 16385, 33001, 65537, 131073, 262145, 300001]


@CUDA
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("vocab", SIZES)
def test_every_vocabulary_size(vocab, dtype):
    hard = (0.0, 0.3)[vocab % 2]
    k = min(vocab, (3, 16, 64)[vocab % 3])
    _check(*_case(4, vocab, k, dtype, vocab, hard, weighted=vocab % 2 == 0), (1.0, 2.0)[vocab % 2], hard)


@CUDA
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("k", [1, 31, 32, 33, 64, 128])
@pytest.mark.parametrize("vocab", [200, 3000])
def test_number_of_entries(k, vocab, dtype):
    _check(*_case(5, vocab, k, dtype, k, 0.5, weighted=True), 1.5, 0.5)


@CUDA
@pytest.mark.parametrize("vocab", [40, 300, 5000])
@pytest.mark.parametrize("hard", [0.0, 0.25, 1.0])
def test_repeated_ids(vocab, hard):
    """An id that a list holds several times counts with the sum of its probabilities."""
    x, ids, teacher, labels, weights = _case(6, vocab, 40 if vocab == 40 else 64, F32, 3, hard)
    ids[0] = 7
    ids[1, ::2] = 11
    ids[2, 5:9] = ids[2, 4]
    ids[3, -1] = ids[3, 0]
    if labels is not None:
        labels[0], labels[1] = 7, 11
    _check(x, ids, teacher, labels, weights, 2.0, hard)


@CUDA
@pytest.mark.parametrize("vocab", [256, 3001, 40000])
def test_rows_that_contribute_nothing(vocab):
    """Weight 0, or neither entries nor label: exactly 0, even on rows without a distribution."""
    from mamba3_b200 import distill as D

    x, ids, teacher, labels, _ = _cuda(*_case(6, vocab, 8, F32, 1, 0.5))
    weights = torch.ones(6, device="cuda")
    weights[0] = 0.0
    ids[1], labels[1] = -1, -100
    x[0], x[1] = math.nan, -math.inf
    ids[2], labels[2] = -1, 3      # the label alone
    labels[3] = -1                 # the entries alone
    ids[0, 0] = vocab + 5          # not looked at: its row has no weight
    loss, dx = D.distill_loss_and_grad(x, ids, teacher, labels=labels, hard_weight=0.5, weights=weights)
    assert torch.isfinite(loss) and torch.isfinite(dx).all()
    assert not dx[:2].any() and dx[2:].any(1).all()
    rows = D.distill_loss(x, ids, teacher, labels=labels, hard_weight=0.5, weights=weights, reduction="none")
    assert not rows[:2].any()
    keep = torch.arange(2, 6)
    cpu = [t.cpu()[keep] for t in (x, ids, teacher, labels)]
    want = R.distill_rows(cpu[0].double(), *cpu[1:], None, 1.0, 0.5)
    assert float((rows[2:].cpu().double() - want).abs().max()) < 5e-5


@CUDA
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("vocab", [256, 3001, 40000])
def test_masked_logits(vocab, dtype):
    """-inf and the type's lowest value in the student's logits, -inf in the teacher's."""
    x, ids, teacher, labels, weights = _case(5, vocab, 16, dtype, 2, 0.3)
    ids = ids.abs() % vocab
    x[0, vocab // 2:] = -math.inf
    ids[0] = ids[0] % (vocab // 2)
    x[1, ::2] = torch.finfo(dtype).min
    ids[1] = torch.arange(16) * 2 + 1
    x[2] = torch.finfo(dtype).min       # uniform
    teacher[3, 4:] = -math.inf          # the rest of the list has probability 0 ...
    x[3, ids[3, 4]] = -math.inf         # ... so that the student may rule it out
    labels[:4] = torch.stack([ids[r, 0] for r in range(4)])
    _check(x, ids, teacher, labels, weights, 1.0, 0.3)


@CUDA
@pytest.mark.parametrize("vocab", [300, 20000])
def test_bad_ids_and_rows_without_a_distribution_show(vocab):
    from mamba3_b200 import distill as D

    x, ids, teacher, labels, _ = _cuda(*_case(5, vocab, 8, BF, 4, 0.5))
    ids = ids.abs()
    labels[:] = 1
    ids[0, 3] = vocab
    labels[1] = 2**33
    x[2] = -math.inf
    x[3, 0] = math.nan
    rows = D.distill_loss(x, ids, teacher, labels=labels, hard_weight=0.5, reduction="none")
    assert torch.isnan(rows[:4]).all() and torch.isfinite(rows[4])
    _, dx = D.distill_loss_and_grad(x, ids, teacher, labels=labels, hard_weight=0.5)
    assert torch.isnan(dx[:4]).all() and torch.isfinite(dx[4]).all()


@CUDA
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("vocab", [250, 256, 2500, 50257])
def test_views_and_in_place(vocab, dtype):
    from mamba3_b200 import distill as D

    x, ids, teacher, labels, weights = _cuda(*_case(12, vocab, 9, dtype, 6, 0.4, weighted=True))
    args = dict(temperature=2.0, hard_weight=0.4)
    loss, dx = D.distill_loss_and_grad(x, ids, teacher, labels=labels, weights=weights, **args)
    buf = torch.full((3, 5, vocab + 13), 77.0, device="cuda", dtype=dtype)
    view = buf[:, 1:, 5:5 + vocab]
    view.copy_(x.view(3, 4, vocab))
    side = [t.view(3, 4, *t.shape[1:]) for t in (ids, teacher, labels, weights)]
    l2, d2 = D.distill_loss_and_grad(view, side[0], side[1], labels=side[2], weights=side[3], **args)
    l3, d3 = D.distill_loss_and_grad(view, side[0], side[1], labels=side[2], weights=side[3], out=view, **args)
    # another split of the row over lanes: the sums may differ in the last bit
    for l, d in ((l2, d2), (l3, d3)):
        assert d.shape == (3, 4, vocab) and abs(float(l) - float(loss)) <= 1e-5 * abs(float(loss))
        assert float((d.reshape(12, vocab).float() - dx.float()).abs().max()) <= 2.0 ** -8 * float(dx.float().abs().max())
    assert torch.equal(d2, d3) and d3.data_ptr() == view.data_ptr()
    assert (buf[:, 0] == 77).all() and (buf[..., :5] == 77).all() and (buf[..., 5 + vocab:] == 77).all()


@CUDA
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,vocab,k,hard", [(60001, 256, 16, 0.0), (20003, 250, 40, 0.4), (2500, 4001, 9, 0.0),
                                               (2500, 2000, 33, 0.4), (2400, 1500, 8, 0.4), (700, 33001, 12, 0.0),
                                               (500, 16390, 64, 0.4)])
def test_many_rows(rows, vocab, k, hard, dtype):
    """Several rows per warp, a row per warp of every length, rows of one, two and more tiles of a CTA."""
    from mamba3_b200 import distill as D

    g = torch.Generator(device="cuda").manual_seed(rows)
    x = (torch.randn(rows, vocab, generator=g, device="cuda") * 2).to(dtype)
    step = vocab // k
    ids = (torch.randint(0, vocab, (rows, 1), generator=g, device="cuda") + torch.arange(k, device="cuda") * step) % vocab
    teacher = torch.randn(rows, k, generator=g, device="cuda") * 2
    ids[:, k // 2][torch.rand(rows, generator=g, device="cuda") < 0.3] = -1
    ids[7], ids[rows // 2] = -1, ids[rows // 2, 0].item()  # no entry; one id k times
    weights = (torch.rand(rows, generator=g, device="cuda") < 0.9).float()
    weights[0] = 1.0
    labels = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.5, ids[:, 0], 3) if hard else None
    T = 1.7
    loss, dx = D.distill_loss_and_grad(x, ids, teacher, temperature=T, labels=labels, hard_weight=hard, weights=weights)
    # the formulas in 64 bits, all rows at once
    there = ids >= 0
    t = torch.where(there, teacher.double() / T, -math.inf)
    p = torch.nan_to_num(torch.softmax(t, 1))
    logq = torch.log_softmax(x.double() / T, 1)
    entries = p * (torch.log(p) - logq.gather(1, ids.clamp_min(0)))
    rows_loss = (1 - hard) * T * T * torch.where(p > 0, entries, 0.0).sum(1)
    soft = there.any(1).double()[:, None]
    grad = (1 - hard) * T * soft * torch.exp(logq)
    grad.scatter_add_(1, ids.clamp_min(0), -(1 - hard) * T * p)
    if hard:
        on = (labels >= 0).double()
        logq1 = torch.log_softmax(x.double(), 1)
        rows_loss = rows_loss - hard * on * logq1.gather(1, labels.clamp_min(0)[:, None])[:, 0]
        hot = torch.zeros_like(grad).scatter_(1, labels.clamp_min(0)[:, None], 1.0)
        grad = grad + hard * on[:, None] * (torch.exp(logq1) - hot)
    w = weights.double()
    grad = grad * (w / w.sum())[:, None]
    assert abs(float(loss) - float((rows_loss * w).sum() / w.sum())) <= _loss_tol(T, x, 1.0)
    _check_grad(dx, grad.cpu(), (w / w.sum() * T)[:, None].cpu(), dtype, "many")
    again, inplace = D.distill_loss_and_grad(x, ids, teacher, temperature=T, labels=labels, hard_weight=hard,
                                             weights=weights, out=x)
    assert inplace is x and torch.equal(again, loss) and torch.equal(x, dx)


@CUDA
def test_gradient_against_differences():
    """Directional differences of the kernel's own loss (fp32, central, step h): rounding of the
    loss 1e-6 / h, truncation h^2 |d3| / 6 with third derivatives of a softmax below 1."""
    from mamba3_b200 import distill as D

    x, ids, teacher, labels, weights = _cuda(*_case(4, 700, 12, F32, 5, 0.3, weighted=True))
    args = dict(temperature=1.3, labels=labels, hard_weight=0.3, weights=weights)
    _, dx = D.distill_loss_and_grad(x, ids, teacher, **args)
    g = torch.Generator().manual_seed(1)
    for _ in range(5):
        d = torch.randn(4, 700, generator=g).cuda()
        h = 3e-3
        up, down = (float(D.distill_loss(x + s * h * d, ids, teacher, **args)) for s in (1, -1))
        assert abs((up - down) / (2 * h) - float((dx * d).sum())) < 2e-6 / h + h * h * 30


@CUDA
def test_same_result_every_call_and_other_streams():
    from mamba3_b200 import distill as D

    x, ids, teacher, labels, weights = _cuda(*_case(64, 9001, 32, BF, 5, 0.3, weighted=True))
    ids[3] = 5  # repeated ids too
    args = dict(temperature=2.0, labels=labels, hard_weight=0.3, weights=weights)
    l1, d1 = D.distill_loss_and_grad(x, ids, teacher, **args)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        l2, d2 = D.distill_loss_and_grad(x + 0, ids, teacher, **args)
    side.synchronize()
    assert torch.equal(l1, l2) and torch.equal(d1, d2)


@CUDA
def test_backward_twice_and_grad_scale():
    from mamba3_b200 import distill as D

    x, ids, teacher, _, _ = _cuda(*_case(8, 600, 6, F32, 5))
    leaf = x.clone().requires_grad_(True)
    loss = D.distill_loss(leaf, ids, teacher)
    a, = torch.autograd.grad(loss, leaf, retain_graph=True)
    b, = torch.autograd.grad(loss, leaf)
    assert torch.equal(a, b)
    _, c = D.distill_loss_and_grad(x, ids, teacher, grad_scale=4.0)
    assert torch.equal(c, 4.0 * a)  # a power of two: exact


@CUDA
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("vocab", [300, 5000])
def test_upstream_of_one_and_others(vocab, weighted, reduction):
    """The gradient that came with the loss, and the ones written in the backward, whatever was done to
    the first in between."""
    from mamba3_b200 import distill as D

    x, ids, teacher, labels, weights = _cuda(*_case(9, vocab, 6, BF, 2, 0.3, weighted=weighted))
    args = dict(labels=labels, hard_weight=0.3, weights=weights, temperature=1.5)
    leaf = x.clone().requires_grad_(True)
    loss = D.distill_loss(leaf, ids, teacher, reduction=reduction, **args)
    one = torch.ones_like(loss)
    first, = torch.autograd.grad(loss, leaf, one, retain_graph=True)
    keep = first.clone()
    first.fill_(5.0)
    again, = torch.autograd.grad(loss, leaf, one, retain_graph=True)
    twice, = torch.autograd.grad(loss, leaf, 2.0 * one, retain_graph=True)
    zero, = torch.autograd.grad(loss, leaf, 0.0 * one)
    assert torch.equal(again, keep) and torch.equal(twice, 2.0 * keep) and not zero.any()
    fresh = x.clone().requires_grad_(True)
    other, = torch.autograd.grad(D.distill_loss(fresh, ids, teacher, reduction=reduction, **args), fresh, 2.0 * one)
    assert torch.equal(other, 2.0 * keep)
    if reduction != "none":
        l2, dx = D.distill_loss_and_grad(x, ids, teacher, reduction=reduction, **args)
        assert torch.equal(dx, keep) and torch.equal(l2, loss.detach())


@CUDA
def test_no_rows():
    from mamba3_b200 import distill as D

    e = torch.empty(0, 5, 30, device="cuda")
    loss, dx = D.distill_loss_and_grad(e, torch.empty(0, 5, 3, dtype=torch.int64, device="cuda"),
                                       torch.empty(0, 5, 3, device="cuda"), reduction="sum")
    assert float(loss) == 0.0 and dx.shape == (0, 5, 30)
    assert D.distill_loss(e, torch.empty(0, 5, 3, dtype=torch.int64, device="cuda"),
                          torch.empty(0, 5, 3, device="cuda"), reduction="none").shape == (0, 5)


@CUDA
def test_refusals():
    from mamba3_b200 import distill as D

    x = torch.zeros(4, 10, device="cuda")
    ids = torch.zeros(4, 3, dtype=torch.int64, device="cuda")
    t = torch.zeros(4, 3, device="cuda")
    lab = torch.zeros(4, dtype=torch.int64, device="cuda")
    wide = torch.zeros(4, 24, device="cuda")
    D.distill_loss_and_grad(wide[:, :10], ids, t, out=wide[:, 11:21])  # columns of one buffer that do not meet
    for bad in (lambda: D.distill_loss(x, ids[:3], t[:3]), lambda: D.distill_loss(x, ids, t[:, :2]),
                lambda: D.distill_loss(x, ids.float(), t), lambda: D.distill_loss(x, ids, ids),
                lambda: D.distill_loss(x, ids, t, temperature=0.0), lambda: D.distill_loss(x, ids, t, hard_weight=0.5),
                lambda: D.distill_loss(x, ids, t, labels=lab), lambda: D.distill_loss(x, ids, t, reduction="max"),
                lambda: D.distill_loss(x, ids, t, hard_weight=1.5, labels=lab),
                lambda: D.distill_loss(x, ids, t, weights=torch.ones(3, device="cuda")),
                lambda: D.distill_loss(x, ids[:, :0], t[:, :0]), lambda: D.distill_loss(x.double(), ids, t),
                lambda: D.distill_loss(x, ids.repeat(1, 50), t.repeat(1, 50)), lambda: D.distill_loss(x.cpu(), ids, t),
                lambda: D.distill_loss_and_grad(x, ids, t, reduction="none"),
                lambda: D.distill_loss_and_grad(x, ids, t, out=torch.empty(4, 11, device="cuda")),
                lambda: D.distill_loss_and_grad(x, ids, t, out=torch.empty(1, 10, device="cuda").expand(4, 10)),
                lambda: D.distill_loss_and_grad(x, ids, t, out=torch.empty(10, 4, device="cuda").t()),
                lambda: D.distill_loss_and_grad(wide[:, :10], ids, t, out=wide[:, 3:13]),
                lambda: D.distill_loss_and_grad(wide[:, :10], ids, t, out=wide.view(-1)[5:45].view(4, 10)),
                lambda: D.distill_loss(x, ids, t, temperature=math.inf)):
        with pytest.raises(ValueError):
            bad()


def test_entry_point_checks_its_arguments():
    from mamba3_b200 import _capi as C

    a = C.M3DistillArgs()
    f = C.lib().m3_distill
    assert f(None, None) == C.M3_ERR_ARG
    assert f(a, None) == C.M3_ERR_SHAPE
    a.rows_outer, a.rows_inner, a.vocab, a.k, a.temperature = 1, 1, 10, 3, 1.0
    assert f(a, None) == C.M3_ERR_ARG  # no logits
    a.k = 129
    assert f(a, None) == C.M3_ERR_SHAPE
    a.k, a.temperature = 3, 0.0
    assert f(a, None) == C.M3_ERR_ARG
    a.temperature, a.logits_dtype = 1.0, 5
    assert f(a, None) == C.M3_ERR_UNSUPPORTED
    a.logits_dtype, a.reduction = 0, 7
    assert f(a, None) == C.M3_ERR_ARG
    a.reduction, a.logits, a.ids, a.teacher, a.row_loss, a.hard_weight = 0, 16, 16, 16, 16, 0.5
    assert f(a, None) == C.M3_ERR_ARG  # no labels
    a.hard_weight, a.ready = 0.0, C.M3_READY_GRAD
    assert f(a, None) == C.M3_ERR_ARG  # a ready gradient without a gradient
    a.ready, a.row_loss = 0, None
    assert f(a, None) == C.M3_ERR_ARG  # neither losses nor a gradient
