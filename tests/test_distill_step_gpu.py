"""The vocabulary-end operators together: a teacher's scores (`train.score`) as the targets of a
student's step (`train.make_distill_step`)."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _model(vocab=300, seed=0, dtype=torch.float32):
    from mamba3_b200 import layer as LY
    from mamba3_b200 import model as M

    cfg = M.LMConfig(vocab_size=vocab, n_layers=2, siso=LY.SISOConfig(d_model=64, d_state=16, headdim=16, chunk=64,
                                                                      policy_name="f32"))
    return cfg, M.init_lm(cfg, seed, dtype=dtype)


def test_score_matches_the_model():
    from mamba3_b200 import model as M
    from mamba3_b200 import train as TR

    cfg, params = _model()
    g = torch.Generator().manual_seed(1)
    xs = torch.randint(0, 300, (2, 128), generator=g).cuda()
    ys = torch.roll(xs, -1, 1)
    ys[:, -1] = -100
    r = TR.score(params, cfg, xs, ys, top=6)
    with torch.no_grad():
        lp = torch.log_softmax(M.lm_forward(params, xs, cfg).double(), -1)
    want = torch.where(ys < 0, 0.0, lp.gather(-1, ys.clamp_min(0)[..., None])[..., 0])
    assert float((r.logprob.double() - want).abs().max()) < 1e-4
    assert float((r.top_logprob.double() - lp.topk(6, -1).values).abs().max()) < 1e-4
    assert float((r.entropy.double() + (lp.exp() * lp).sum(-1)).abs().max()) < 1e-4


def test_gradients_match_torch_and_the_student_learns():
    from mamba3_b200 import model as M
    from mamba3_b200 import train as TR

    cfg, teacher = _model(seed=3)
    teacher = teacher._replace(embed=teacher.embed * 8)  # a teacher with something to say
    _, student = _model(seed=4)
    g = torch.Generator().manual_seed(2)
    xs = torch.randint(0, 300, (2, 128), generator=g).cuda()
    ys = torch.randint(0, 300, (2, 128), generator=g).cuda()
    ref = TR.score(teacher, cfg, xs, top=20)
    weights = (torch.rand(2, 128, generator=g) < 0.9).float().cuda()

    # the same loss written in torch
    leaves = TR.param_list(student)
    for p in leaves:
        p.requires_grad_(True)
    logits = M.lm_forward(student, xs, cfg, compute_dtype=torch.float32)
    p = torch.softmax(ref.top_logprob / 2.0, -1)
    q = torch.log_softmax(logits / 2.0, -1).gather(-1, ref.top_ids)
    rows = 0.7 * 4.0 * (p * (p.log() - q)).sum(-1) + 0.3 * torch.nn.functional.cross_entropy(
        logits.reshape(-1, 300), ys.reshape(-1), reduction="none").view(2, 128)
    loss = (rows * weights).sum() / weights.sum()
    want = torch.autograd.grad(loss, leaves)

    grads = {}
    step = TR.make_distill_step(cfg, student, temperature=2.0, hard_weight=0.3, lr=3e-3, clip=None,
                                compute_dtype=torch.float32, distributed=False)
    update = step.optimizer.step
    step.optimizer.step = lambda: (grads.update({i: t.grad.clone() for i, t in enumerate(step.params)}), update())
    first = float(step(xs, ref.top_ids, ref.top_logprob, ys, weights))
    step.optimizer.step = update
    assert abs(first - float(loss)) < 1e-4
    for i, w in enumerate(want):
        assert float((grads[i] - w).norm() / w.norm().clamp_min(1e-12)) < 1e-3, i
    for _ in range(15):
        last = float(step(xs, ref.top_ids, ref.top_logprob, ys, weights))
    assert last < 0.9 * first


def test_padding_tokens():
    from mamba3_b200 import train as TR

    cfg, teacher = _model(seed=3)
    _, student = _model(seed=4)
    xs = torch.randint(0, 300, (1, 64), generator=torch.Generator().manual_seed(5)).cuda()
    ref = TR.score(teacher, cfg, xs, top=4)
    xs[0, 60:] = -1
    weights = (xs >= 0).float()
    step = TR.make_distill_step(cfg, student, compute_dtype=torch.bfloat16, distributed=False)
    assert torch.isfinite(step(xs, ref.top_ids, ref.top_logprob, weights=weights))
