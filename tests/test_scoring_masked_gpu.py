"""`scoring.token_logprobs` on rows of which a mask leaves only a few ids (constrained decoding), by a cluster, a
CTA or a warp a row, one or many of them: fewer ids than alternatives, or somewhat more.

Tolerances as in test_scoring_gpu: ln Z to 4e-6 and 3e-7 of the logits' size (at most 20 here); a log probability
of the lowest value of the type to a few roundings (1e-6 of it)."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lowest", [False, True])
@pytest.mark.parametrize("rows,vocab", [(5, 128256), (160, 128256), (400, 20011), (2500, 4001), (3000, 700), (9000, 256)])
@pytest.mark.parametrize("left,top", [(10, 20), (100, 20), (100, 64), (1, 1)])
def test_few_ids_left(rows, vocab, left, top, lowest, dtype):
    from mamba3_b200 import scoring as S

    g = torch.Generator(device="cuda").manual_seed(vocab + left)
    mask = torch.finfo(dtype).min if lowest else -math.inf
    x = torch.full((rows, vocab), mask, dtype=dtype, device="cuda")
    ids = (torch.randint(0, vocab, (rows, 1), generator=g, device="cuda") +
           torch.arange(left, device="cuda") * (1 + torch.randint(0, vocab // left, (rows, 1), generator=g, device="cuda"))) % vocab
    x.scatter_(1, ids, (torch.randn(rows, left, generator=g, device="cuda") * 3).to(dtype))
    t = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.8, ids[:, -1], 0)
    got = S.token_logprobs(x, t, top=top, temperature=0.9)
    y = x.double() / 0.9
    d = y - y.amax(1, keepdim=True)
    ln_z = torch.log(torch.exp(d).sum(1))
    lp = d - ln_z[:, None]
    p = torch.exp(lp)
    atol = 4e-6 + 3e-7 * 20
    order = torch.sort(x.float() + 0.0, dim=1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(got.top_ids, order)
    for have, want, tol in ((got.lse, y.amax(1) + ln_z, atol), (got.entropy, -torch.where(p > 0, p * lp, 0.0).sum(1), 8 * atol),
                            (got.logprob, lp.gather(1, t[:, None])[:, 0], atol), (got.top_logprob, lp.gather(1, order), atol)):
        want = want.float()  # past fp32: -inf
        assert torch.equal(torch.isinf(have), torch.isinf(want)) and not torch.isnan(have).any()
        ok = torch.isfinite(want)
        assert ((have - want)[ok].abs() <= tol + 1e-6 * want[ok].abs()).all()
