"""`scoring.token_logprobs` against the 64-bit formulas: vocabularies around every size at which
the kernel changes its split, views, masked logits, ties, rows without a distribution.

Tolerances, from the arithmetic (fp32, exponent arguments below ~30 in log2 units where they
matter): an exponential is off by 2^-22 + 30 * 2^-24 relative, so ln Z by < 3e-6 absolute; the
row maximum and the result are rounded at their own size (2^-23 relative each); the entropy adds
a sum weighted by d <= ln V."""

import math

import pytest
import torch

from tests import vocab_ref as R

CUDA = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _close(got, want, atol, rtol, what):
    got, want = got.double().cpu(), want.double()
    assert got.shape == want.shape, what
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), what
    ok = torch.isfinite(want)
    err = (got[ok] - want[ok]).abs() - rtol * want[ok].abs()
    assert err.numel() == 0 or float(err.max()) <= atol, (what, float(err.max()))


def _check(logits, targets, top, temperature):
    from mamba3_b200 import scoring as S

    got = S.token_logprobs(logits, targets, top=top, temperature=temperature)
    flat = logits.reshape(-1, logits.shape[-1]).cpu()
    want = R.score(flat, None if targets is None else targets.reshape(-1).cpu(), top, temperature)
    lead = logits.shape[:-1]
    size = float(torch.nan_to_num(flat.float(), posinf=0.0, neginf=0.0).abs().clamp(max=1e30).max()) / temperature
    atol = 4e-6 + 3e-7 * min(size, 1e4)
    _close(got.lse, want["lse"].view(lead), atol, 1e-6, "lse")
    _close(got.entropy, want["entropy"].view(lead), 8 * atol, 1e-6, "entropy")
    if targets is None:
        assert got.logprob is None
    else:
        _close(got.logprob, want["logprob"].view(lead), atol, 1e-6, "logprob")
    if top:
        assert torch.equal(got.top_ids.cpu(), want["top_ids"].view(*lead, top))
        _close(got.top_logprob, want["top_logprob"].view(*lead, top), atol, 1e-6, "top_logprob")
    else:
        assert got.top_ids is None and got.top_logprob is None


def _logits(shape, dtype, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * spread).to(dtype).cuda()


def _targets(lead, vocab, seed):
    g = torch.Generator().manual_seed(seed + 1)
    t = torch.randint(0, vocab, lead, generator=g)
    t[torch.rand(lead, generator=g) < 0.2] = -100
    return t.cuda()


SIZES = [1, 2, 7, 31, 32, 255, 256, 257, 511, 512, 513, 1000, 1024, 1025, 2047, 2049, 4096, 4099, 8191, 8193, 16385,
         32768, 33000, 65537, 100003, 131073, 262145, 300000]


@CUDA
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("vocab", SIZES)
def test_every_vocabulary_size(vocab, dtype):
    rows = 3
    top = min(vocab, (5, 20, 128)[vocab % 3])
    _check(_logits((rows, vocab), dtype, vocab), _targets((rows,), vocab, vocab), top, 1.0)


@CUDA
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,vocab", [(1, 128256), (2, 5000), (700, 300), (400, 9001), (333, 520)])
@pytest.mark.parametrize("top", [0, 1, 8])
def test_row_counts(rows, vocab, top, dtype):
    _check(_logits((rows, vocab), dtype, rows), _targets((rows,), vocab, rows), top, 0.7)


@CUDA
@pytest.mark.parametrize("k", [1, 2, 31, 32, 33, 64, 127, 128])
@pytest.mark.parametrize("vocab", [128, 256, 700, 5000, 70001])
def test_number_of_alternatives(k, vocab):
    _check(_logits((2, vocab), BF, k), None, k, 2.0)  # bf16: many exact ties


@CUDA
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("vocab", [250, 256, 5001, 50257])
def test_shifted_and_padded_views(vocab, dtype):
    """logits[:, :-1] of a padded head against tokens[:, 1:]: two strides, rows of any alignment."""
    buf = _logits((3, 6, vocab + 47), dtype, 5)
    tokens = _targets((3, 6), vocab, 5)
    _check(buf[:, :-1, :vocab], tokens[:, 1:], 7, 1.0)
    _check(buf[:, 1:, 3:vocab], tokens.to(torch.int32)[:, :-1].clamp(max=vocab - 4), 7, 1.0)
    _check(buf.transpose(0, 1)[..., :vocab], None, 3, 1.0)
    _check(buf[..., 1:2 * (vocab // 2):2], None, 3, 1.0)  # a strided vocabulary axis is copied
    _check(buf[0, 0, :vocab], torch.tensor(4, device="cuda"), 2, 1.0)  # one row, no leading axes
    _check(buf[0, :1, :vocab].expand(4, vocab), None, 2, 1.0)


@CUDA
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("vocab", [64, 256, 3001, 40000])
def test_masked_and_tied_rows(vocab, dtype):
    x = _logits((12, vocab), dtype, 9)
    low = torch.finfo(dtype).min
    x[0] = -math.inf                      # nothing left: NaN, ids in order
    x[1] = low                            # everything at the lowest value: uniform
    x[2, 1:] = -math.inf                  # one id left: entropy 0
    x[3, ::2] = -math.inf
    x[4] = 1.5                            # all equal
    x[5, :] = low
    x[5, vocab // 2] = 0.0                # one id above a mask of the lowest value
    x[6, vocab - 1] = math.inf
    x[7, vocab // 3] = math.nan
    x[8] = torch.where(torch.arange(vocab, device="cuda") % 2 == 0, 0.0, -0.0).to(dtype)  # -0 == +0
    x[9] = torch.arange(vocab, device="cuda").to(dtype)   # the largest side by side
    x[10, : vocab // 2] = math.nan
    x[11] = torch.finfo(dtype).max / 4
    t = torch.full((12,), vocab // 2, device="cuda")
    t[3] = 0                              # a masked target: -inf
    _check(x, t, min(vocab, 40), 1.0)
    _check(x, t, min(vocab, 128), 1.0)


@CUDA
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("vocab", [64, 256, 3001, 40000])
def test_suppressed_ids(vocab, dtype):
    """-inf masks over logits of ordinary size (and so at the tolerance of ordinary rows)."""
    x = _logits((6, vocab), dtype, 4)
    x[0, 1:] = -math.inf
    x[1, ::2] = -math.inf
    x[2, : vocab - 3] = -math.inf
    x[3, 8:] = -math.inf
    x[4, torch.arange(vocab, device="cuda") % 16 != 5] = -math.inf
    _check(x, torch.full((6,), vocab - 1, device="cuda"), min(vocab, 12), 1.3)


def _vector_reference(x, t, temperature):
    """The formulas in 64 bits over all rows at once (on the device): rows with a finite maximum."""
    y = x.double() / temperature
    d = y - y.amax(-1, keepdim=True)
    z = torch.exp(d).sum(-1)
    lp = d - torch.log(z)[:, None]
    p = torch.exp(lp)
    ent = -torch.where(p > 0, p * lp, 0.0).sum(-1)
    picked = torch.where(t < 0, 0.0, lp.gather(1, t.clamp_min(0)[:, None])[:, 0])
    return picked, ent, y.amax(-1) + torch.log(z), lp


@CUDA
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,vocab,top", [(60001, 256, 8), (60001, 250, 3), (20003, 300, 20), (2500, 4001, 8),
                                            (2500, 4001, 32), (2500, 2000, 0), (2400, 8100, 5), (19000, 520, 40),
                                            (700, 33001, 12)])
def test_many_rows(rows, vocab, top, dtype):
    """Several rows per warp, one warp per longer row, several waves of CTAs; masks and ties among them."""
    from mamba3_b200 import scoring as S

    x = _logits((rows, vocab), dtype, rows + vocab)
    x[:, 5] = -math.inf
    x[rows // 3] = 0.25
    x[rows // 2, 1::2] = -math.inf
    x[rows - 1] = torch.arange(vocab, device="cuda").to(dtype) / 16
    t = _targets((rows,), vocab, 3)
    got = S.token_logprobs(x, t, top=top, temperature=1.2)
    picked, ent, lse, lp = _vector_reference(x, t, 1.2)
    tol = 4e-6 + 3e-7 * float(x[:, 6:].float().abs().clamp(max=1e4).max()) / 1.2
    _close(got.lse, lse.cpu(), tol, 1e-6, "lse")
    _close(got.entropy, ent.cpu(), 8 * tol, 1e-6, "entropy")
    _close(got.logprob, picked.cpu(), tol, 1e-6, "logprob")
    if top:
        # ties to the lower index: an order of all entries that is stable in the index
        order = torch.sort(x.float() + 0.0, dim=1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(got.top_ids, order)
        _close(got.top_logprob, lp.gather(1, order).cpu(), tol, 1e-6, "top_logprob")


@CUDA
@pytest.mark.parametrize("temperature", [1e-12, 1e-6, 1e-3, 50.0, 1e6, 1e12])
@pytest.mark.parametrize("vocab", [200, 3000])
def test_temperatures(vocab, temperature):
    """From a distribution on one id to a uniform one; both forms of the sums."""
    from mamba3_b200 import scoring as S

    x = _logits((6, vocab), F32, 2)
    x[1, ::3] = -math.inf
    got = S.token_logprobs(x, None, top=3, temperature=temperature)
    _, ent, lse, lp = _vector_reference(x, torch.zeros(6, dtype=torch.int64, device="cuda"), temperature)
    top = lp.topk(3, 1).values
    _close(got.lse, lse.cpu(), 1e-5, 1e-6, "lse")
    _close(got.entropy, ent.cpu(), 5e-5, 1e-6, "entropy")
    _close(got.top_logprob, top.cpu(), 1e-5, 2e-6, "top_logprob")


@CUDA
def test_targets_outside_the_vocabulary():
    from mamba3_b200 import scoring as S

    x = _logits((5, 100), BF, 1)
    t = torch.tensor([-1, 0, 99, 100, 2**40], device="cuda")
    lp = S.token_logprobs(x, t).logprob.cpu()
    assert float(lp[0]) == 0.0 and torch.isfinite(lp[1:3]).all() and torch.isnan(lp[3:]).all()


@CUDA
def test_no_rows_and_same_result_every_call():
    from mamba3_b200 import scoring as S

    r = S.token_logprobs(torch.empty(0, 4, 77, device="cuda"), torch.empty(0, 4, dtype=torch.int64, device="cuda"), top=3)
    assert r.logprob.shape == (0, 4) and r.top_ids.shape == (0, 4, 3)
    r = S.token_logprobs(torch.empty(4, 0, 77, device="cuda"))
    assert r.lse.shape == (4, 0)
    x = _logits((300, 9000), BF, 3)
    a, b = (S.token_logprobs(x, None, top=50) for _ in range(2))
    assert all(torch.equal(u, v) for u, v in zip(a[1:], b[1:]))


@CUDA
def test_other_streams():
    from mamba3_b200 import scoring as S

    x = _logits((64, 30000), BF, 3)
    want = S.token_logprobs(x, top=4)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y = x + 0
        got = S.token_logprobs(y, top=4)
    side.synchronize()
    assert torch.equal(got.lse, want.lse) and torch.equal(got.top_ids, want.top_ids)


@CUDA
def test_replayed_in_a_graph():
    """Captured calls read their inputs anew: scoring, the distillation step and the lookup's gradient."""
    from mamba3_b200 import distill as D
    from mamba3_b200 import embedding as E
    from mamba3_b200 import scoring as S

    x, x2 = _logits((40, 9000), BF, 1), _logits((40, 9000), BF, 2)
    ids = torch.randint(0, 9000, (40, 6), device="cuda")
    teacher = torch.randn(40, 6, device="cuda")
    w = torch.rand(40, device="cuda")
    dy = torch.randn(40, 64, device="cuda")

    def step():
        r = S.token_logprobs(x, ids[:, 0], top=4)
        loss, dx = D.distill_loss_and_grad(x, ids, teacher, weights=w)
        return r.logprob, r.entropy, r.top_ids, loss, dx, E.embedding_grad(dy, ids[:, 1], 9000)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    x.copy_(x2)
    ids.copy_(torch.randint(0, 9000, (40, 6), device="cuda"))
    graph.replay()
    for a, b in zip(got, step()):
        assert torch.equal(a, b)


@CUDA
def test_refusals():
    from mamba3_b200 import scoring as S

    x = torch.zeros(4, 10, device="cuda")
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    for bad in (lambda: S.token_logprobs(x, top=11), lambda: S.token_logprobs(x, top=-1),
                lambda: S.token_logprobs(torch.zeros(2, 500, device="cuda"), top=129),
                lambda: S.token_logprobs(x, temperature=0.0), lambda: S.token_logprobs(x, temperature=math.inf),
                lambda: S.token_logprobs(x, temperature=1e-38), lambda: S.token_logprobs(x, temperature=math.nan),
                lambda: S.token_logprobs(x, t[:3]), lambda: S.token_logprobs(x, t.float()),
                lambda: S.token_logprobs(x.double()), lambda: S.token_logprobs(x, t.cpu()),
                lambda: S.token_logprobs(torch.zeros(3, 0, device="cuda"))):
        with pytest.raises(ValueError):
            bad()


def test_refuses_cpu_tensors():
    from mamba3_b200 import scoring as S

    with pytest.raises(ValueError):
        S.token_logprobs(torch.zeros(2, 5))


def test_entry_point_checks_its_arguments():
    """On the host, before any launch."""
    from mamba3_b200 import _capi as C

    a = C.M3ScoreArgs()
    f = C.lib().m3_token_logprobs
    assert f(None, None) == C.M3_ERR_ARG
    assert f(a, None) == C.M3_ERR_SHAPE  # vocab 0
    a.rows_outer, a.rows_inner, a.vocab, a.temperature = 1, 1, 10, 1.0
    assert f(a, None) == C.M3_ERR_ARG  # no logits
    a.top = 11
    assert f(a, None) == C.M3_ERR_SHAPE
    a.top, a.logits_dtype = 0, 9
    assert f(a, None) == C.M3_ERR_UNSUPPORTED
    a.logits_dtype, a.temperature = 0, -1.0
    assert f(a, None) == C.M3_ERR_ARG
    a.temperature, a.rows_inner = 1.0, 0
    assert f(a, None) == C.M3_OK  # nothing to do
