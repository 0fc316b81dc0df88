"""The vocabulary-end operators at the ends of their ranges: temperatures, rows without weight,
distributions on one entry."""

import math

import pytest
import torch

from tests import vocab_ref as R

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("vocab", [200, 3000, 40000])
@pytest.mark.parametrize("temperature", [2.0 ** -99, 2.0 ** -66, 2.0 ** -40, 2.0 ** -10])
def test_distillation_at_low_temperatures(vocab, temperature):
    """T^2 KL where T^2 is not an fp32 number.  Both distributions are on one entry (logits apart by more than
    2^-10 * 100), so that KL = (x_max - x_id) / T and the loss T (x_max - x_id), to a few roundings (1e-5)."""
    from mamba3_b200 import distill as D

    g = torch.Generator().manual_seed(vocab)
    rows, k = 5, 7
    x = torch.stack([torch.randperm(vocab, generator=g) for _ in range(rows)]).float() / 8
    ids = torch.stack([torch.randperm(vocab, generator=g)[:k] for _ in range(rows)])
    teacher = torch.stack([torch.randperm(k, generator=g) for _ in range(rows)]).float()
    xd = x.double().requires_grad_(True)
    want = R.distill_rows(xd, ids, teacher, None, None, temperature, 0.0)
    grad, = torch.autograd.grad(want.sum(), xd)
    args = (x.cuda(), ids.cuda(), teacher.cuda())
    got = D.distill_loss(*args, temperature=temperature, reduction="none").double().cpu()
    assert (want > 0).all()
    assert ((got - want).abs() <= 1e-5 * want.abs()).all()
    loss, dx = D.distill_loss_and_grad(*args, temperature=temperature, reduction="sum")
    assert abs(float(loss) - float(want.sum())) <= 1e-5 * float(want.sum())
    assert ((dx.double().cpu() - grad).abs() <= 1e-5 * grad.abs() + 1e-40).all()  # 1e-40: below fp32


@pytest.mark.parametrize("vocab", [200, 40000])
def test_distillation_at_high_temperatures(vocab):
    from mamba3_b200 import distill as D

    g = torch.Generator().manual_seed(vocab)
    x, teacher = torch.randn(4, vocab, generator=g).cuda(), torch.randn(4, 6, generator=g).cuda()
    ids = torch.randint(0, vocab, (4, 6), generator=g).cuda()
    for t in (1e19, 1e30):  # T^2 is past fp32
        with pytest.raises(ValueError):
            D.distill_loss(x, ids, teacher, temperature=t)
        with pytest.raises(ValueError):
            D.distill_loss_and_grad(x, ids, teacher, temperature=t)
    loss, dx = D.distill_loss_and_grad(x, ids, teacher, temperature=1e18)
    assert torch.isfinite(loss) and torch.isfinite(dx).all()


@pytest.mark.parametrize("vocab", [256, 3001, 40000])
@pytest.mark.parametrize("hard", [0.0, 0.5])
def test_mean_over_rows_without_weight(vocab, hard):
    """No row contributes: loss and gradient are 0, as for a single row of weight 0."""
    from mamba3_b200 import distill as D

    x = torch.randn(6, vocab, device="cuda")
    x[1] = math.nan
    ids = torch.randint(0, vocab, (6, 4), device="cuda")
    teacher, weights = torch.randn(6, 4, device="cuda"), torch.zeros(6, device="cuda")
    args = dict(weights=weights, hard_weight=hard, labels=ids[:, 1] if hard else None)
    for reduction in ("mean", "sum"):
        loss, dx = D.distill_loss_and_grad(x, ids, teacher, reduction=reduction, **args)
        assert float(loss) == 0.0 and not dx.any()
        leaf = x.clone().requires_grad_(True)
        loss = D.distill_loss(leaf, ids, teacher, reduction=reduction, **args)
        (2.0 * loss).backward()
        assert float(loss) == 0.0 and not leaf.grad.any()
        with torch.no_grad():
            assert float(D.distill_loss(x, ids, teacher, reduction=reduction, **args)) == 0.0
    weights[2] = 0.5  # a mean over one row
    loss, _ = D.distill_loss_and_grad(x, ids, teacher, **args)
    rows = D.distill_loss(x, ids, teacher, reduction="none", **args)
    assert float(loss) == float(rows[2]) * 2.0
    x[2, 0] = math.nan
    assert torch.isnan(D.distill_loss_and_grad(x, ids, teacher, **args)[0])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("vocab", [1, 2, 200, 700, 5000, 40000, 300000])
def test_probabilities_of_at_most_one(vocab, dtype):
    """Rows on one entry: a log probability is never above 0 nor an entropy below it, and both are within
    the rounding of a sum (|logit| 2^-22) of 0."""
    from mamba3_b200 import scoring as S

    g = torch.Generator().manual_seed(vocab)
    rows, top = 40, min(vocab, 3)
    at = torch.randint(0, vocab, (rows,), generator=g)
    x = torch.full((rows, vocab), -math.inf)
    x[::2] = torch.randn(rows // 2, vocab, generator=g) - 300  # the rest: 2^-300 and less
    x[torch.arange(rows), at] = torch.randn(rows, generator=g) * 20
    x = x.to(dtype)
    x, at = x.cuda(), at.cuda()
    for temperature in (1.0, 0.7, 1.9):
        for k in (0, top):
            r = S.token_logprobs(x, at, top=k, temperature=temperature)
            tol = float(x.max()) / temperature * 2.0 ** -22 + 1e-6
            assert float(r.entropy.min()) >= 0.0 and float(r.entropy.max()) <= tol
            assert float(r.logprob.max()) <= 0.0 and float(r.logprob.min()) >= -tol
            if k:
                assert float(r.top_logprob.max()) <= 0.0 and torch.equal(r.top_ids[:, 0], at)
    x[3, 0] = math.nan
    r = S.token_logprobs(x, at, top=top)
    assert torch.isnan(r.entropy[3]) and torch.isnan(r.logprob[3]) and torch.isfinite(r.entropy[:3]).all()


@pytest.mark.parametrize("rows,vocab", [(5000, 64), (9, 40000), (700, 3000)])
@pytest.mark.parametrize("weighted", [False, True])
def test_losses_of_calls_in_a_row(rows, vocab, weighted):
    """The sum of the rows' losses starts before they are all written and waits for them: calls one behind the
    other, whose workspaces are the same memory, each give their own.  A sum of positive terms in a tree of
    fewer than 40 levels: 40 * 2^-24 relative, and as much for the weights' sum."""
    from mamba3_b200 import distill as D

    g = torch.Generator(device="cuda").manual_seed(rows)
    ids = torch.randint(0, vocab, (rows, 4), generator=g, device="cuda")
    teacher = torch.randn(rows, 4, generator=g, device="cuda")
    xs = [torch.randn(rows, vocab, generator=g, device="cuda") * (1 + i) for i in range(4)]
    ws = [torch.rand(rows, generator=g, device="cuda") + 0.1 if weighted else None for _ in xs]
    losses = [D.distill_loss(xs[i % 4], ids, teacher, weights=ws[i % 4]) for i in range(60)]
    steps = [D.distill_loss_and_grad(xs[i % 4], ids, teacher, weights=ws[i % 4])[0] for i in range(8)]
    for i in range(4):
        per_row = D.distill_loss(xs[i], ids, teacher, weights=ws[i], reduction="none").double()
        want = float(per_row.sum() / (rows if ws[i] is None else ws[i].double().sum()))
        for got in losses[i::4] + steps[i::4]:
            assert abs(float(got) - want) <= 80 * 2.0 ** -24 * want


@pytest.mark.parametrize("upstream", [1.0, 2.0])
@pytest.mark.parametrize("vocab", [64, 3000, 40000])
def test_ready_gradient_without_ready_weights(vocab, upstream):
    """The C entry with a gradient that is there and a weight sum that is not: left alone or written anew."""
    from mamba3_b200 import _capi as C
    from mamba3_b200 import _tensors as T
    from mamba3_b200 import distill as D

    g = torch.Generator(device="cuda").manual_seed(vocab)
    x, teacher = torch.randn(50, vocab, generator=g, device="cuda"), torch.randn(50, 4, generator=g, device="cuda")
    ids, w = torch.randint(0, vocab, (50, 4), generator=g, device="cuda"), torch.rand(50, generator=g, device="cuda") + 0.1
    _, want = D.distill_loss_and_grad(x, ids, teacher, weights=w, grad_scale=upstream)
    grad, up, total = torch.full_like(x, 7.0), torch.full((1,), upstream, device="cuda"), torch.zeros(1, device="cuda")
    a = C.M3DistillArgs(1, 50, vocab, 4, T.io_dtype(x.dtype), C.M3_REDUCE_MEAN, 1.0, 0.0, 1.0, x.data_ptr(), 0, vocab,
                        ids.data_ptr(), teacher.data_ptr(), None, w.data_ptr(), up.data_ptr(), 0, None, None,
                        total.data_ptr(), grad.data_ptr(), 0, vocab, C.M3_READY_GRAD, 0)
    T.call(C.lib().m3_distill, a, x.device)
    after = total.clone()  # behind the call in the stream: behind the sum of weights too
    assert abs(float(after) - float(w.double().sum())) <= 1e-5 * 50
    assert (grad == 7).all() if upstream == 1 else torch.equal(grad, want)
