"""`embedding.embed_tokens` and `embedding_grad` against the 64-bit formulas.

Tolerances: the lookup is one fp32 product and one rounding, so it is exact to the output's own
rounding (half a unit in the last place: 2^-24 or, with bf16's 8-bit significand, 2^-8 relative, plus the product's 2^-24).  A gradient row is a fp32 sum of n
terms: n 2^-24 of the terms' magnitudes, plus its rounding."""

import math

import pytest
import torch

from tests import vocab_ref as R

CUDA = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
EPS = {F32: 2.0 ** -24, BF: 2.0 ** -8}


def _tokens(shape, vocab, seed, skew=False):
    g = torch.Generator().manual_seed(seed)
    t = torch.randint(0, vocab, shape, generator=g)
    if skew:  # most positions share one id
        t = torch.where(torch.rand(shape, generator=g) < 0.7, vocab // 2, t)
    t[torch.rand(shape, generator=g) < 0.1] = -1
    return t


def _rows(shape, dtype, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _check_lookup(table, tokens, scale, dtype):
    from mamba3_b200 import embedding as E

    got = E.embed_tokens(table, tokens, scale=scale, dtype=dtype).cpu()
    want = R.embed(table.cpu(), tokens.cpu(), scale)
    assert got.dtype == dtype and got.shape == want.shape
    bad = torch.isnan(want)
    assert torch.equal(torch.isnan(got), bad)
    err = (got.double() - want).abs() - want.abs() * (EPS[dtype] + 2.0 ** -23)
    assert want[~bad].numel() == 0 or float(err[~bad].max()) <= 0


def _check_grad(dy, tokens, vocab, scale, dtype, out=None):
    from mamba3_b200 import embedding as E

    base = None if out is None else out.double().cpu()
    got = E.embedding_grad(dy, tokens, vocab, scale=scale, dtype=dtype, out=out).double().cpu()
    want = R.embed_grad(dy.cpu(), tokens.cpu(), vocab, scale)
    size = R.embed_grad(dy.abs().cpu(), tokens.cpu(), vocab, abs(scale))
    n = R.embed_grad(torch.ones(*tokens.shape, 1), tokens.cpu(), vocab, 1.0)
    if base is not None:
        assert torch.equal(got[(n == 0)[:, 0]], base[(n == 0)[:, 0]])
        want, size, n = want + base, size + base.abs(), n + 1
    tol = size * (n + 2) * 2.0 ** -24 + want.abs() * EPS[dtype] * 1.01
    assert float(((got - want).abs() - tol).max()) <= 0


@CUDA
@pytest.mark.parametrize("table_dtype,dtype", [(F32, BF), (BF, BF), (BF, F32), (F32, F32)])
@pytest.mark.parametrize("dim", [1, 3, 8, 12, 64, 100, 512, 1025, 2048, 2056, 5000])
def test_lookup(table_dtype, dtype, dim):
    table = _rows((50, dim), table_dtype, dim).cuda()
    _check_lookup(table, _tokens((3, 7), 50, dim).cuda(), 3.7, dtype)
    _check_lookup(table, _tokens((), 50, 1).cuda(), 1.0, dtype)


@CUDA
@pytest.mark.parametrize("dim", [64, 100, 257])
def test_lookup_views_and_ids(dim):
    from mamba3_b200 import embedding as E

    buf = _rows((40, dim + 9), F32, 1).cuda()
    tokens = _tokens((4, 9, 3), 40, 2).cuda()
    _check_lookup(buf[:, 5:5 + dim], tokens[:, 1:, 0], 1.0, BF)   # strided ids, a slice of a wider table
    _check_lookup(buf[:, 1:1 + dim], tokens.to(torch.int32).permute(2, 0, 1), 2.0, F32)
    _check_lookup(buf.t()[:dim + 1, :40], tokens[0, 0] % (dim + 1), 1.0, F32)     # a transposed table is copied
    t = torch.tensor([0, 39, 40, -5, 2**40], device="cuda")
    out = E.embed_tokens(buf, t)
    assert torch.isfinite(out[:2]).all() and torch.isnan(out[[2, 4]]).all() and not out[3].any()
    assert E.embed_tokens(buf, t[:0]).shape == (0, dim + 9)


@CUDA
@pytest.mark.parametrize("dy_dtype,dtype", [(BF, F32), (BF, BF), (F32, F32), (F32, BF)])
@pytest.mark.parametrize("rows,vocab,dim", [(1, 5, 8), (2, 1, 16), (31, 600, 100), (1000, 7, 64), (500, 70000, 8),
                                            (3000, 256, 40), (257, 300, 2049), (4097, 513, 33), (20000, 3, 24)])
def test_gradient(rows, vocab, dim, dy_dtype, dtype):
    dy = _rows((rows, dim), dy_dtype, rows).cuda()
    for skew in (False, True):
        _check_grad(dy, _tokens((rows,), vocab, rows, skew).cuda(), vocab, 1.7, dtype)


@CUDA
@pytest.mark.parametrize("vocab", [2, 511, 512, 513, 2**18 - 1, 2**18 + 1, 300001])
def test_gradient_ids_of_every_width(vocab):
    """One, two and three digits in the sort; the first and the last id occur."""
    t = _tokens((6, 50), vocab, vocab)
    t[0, 0], t[0, 1], t[3, 3] = 0, vocab - 1, vocab - 1
    _check_grad(_rows((6, 50, 16), F32, 3).cuda(), t.cuda(), vocab, 1.0, F32)


@CUDA
@pytest.mark.parametrize("dtype", [BF, F32])
def test_gradient_added_to_another(dtype):
    out = _rows((300, 72), dtype, 1).cuda()
    _check_grad(_rows((5, 40, 72), BF, 2).cuda(), _tokens((5, 40), 300, 3, True).cuda(), 300, 0.5, dtype, out=out)
    wide = _rows((300, 80), dtype, 1).cuda()
    keep = wide.clone()
    _check_grad(_rows((700, 72), BF, 2).cuda(), _tokens((700,), 300, 3).cuda(), 300, 0.5, dtype, out=wide[:, 4:76])
    assert torch.equal(wide[:, :4], keep[:, :4]) and torch.equal(wide[:, 76:], keep[:, 76:])


@CUDA
def test_gradient_views_no_rows_and_ids_outside():
    from mamba3_b200 import embedding as E

    dy = _rows((4, 9, 48), F32, 1).cuda()
    t = _tokens((4, 9), 30, 1).cuda()
    _check_grad(dy[:, 1:, 3:35], t[:, :-1], 30, 1.0, F32)
    _check_grad(dy.transpose(0, 1), t.t(), 30, 1.0, F32)
    _check_grad(dy[:1].expand(4, 9, 48), t, 30, 1.0, F32)
    assert not E.embedding_grad(dy[:0], t[:0], 30).any()
    t[:] = 30  # at or past the table's end, and padding: no gradient
    t[0] = -7
    assert not E.embedding_grad(dy, t, 30).any()
    same = torch.full((30, 48), 2.5, device="cuda")
    assert (E.embedding_grad(dy, t, 30, out=same) == 2.5).all()


@CUDA
def test_autograd_and_differences():
    from mamba3_b200 import embedding as E

    table = _rows((20, 24), F32, 1).cuda().requires_grad_(True)
    t = _tokens((3, 50), 20, 1).cuda()
    dy = _rows((3, 50, 24), F32, 2).cuda()
    out = E.embed_tokens(table, t, scale=1.5)
    out.backward(dy)
    want = R.embed_grad(dy.cpu(), t.cpu(), 20, 1.5)
    assert float((table.grad.double().cpu() - want).abs().max()) < 1e-5
    d = _rows((20, 24), F32, 3).cuda()
    with torch.no_grad():  # linear in the table: a difference is exact but for rounding
        diff = ((E.embed_tokens(table + d, t, scale=1.5) - E.embed_tokens(table - d, t, scale=1.5)) * dy).double().sum() / 2
    assert abs(float(diff) - float((table.grad * d).double().sum())) < 2e-3
    bf = _rows((20, 24), BF, 1).cuda().requires_grad_(True)
    E.embed_tokens(bf, t, dtype=F32).sum().backward()
    assert bf.grad.dtype == BF


@CUDA
def test_same_result_every_call_and_other_streams():
    from mamba3_b200 import embedding as E

    t = _tokens((20000,), 900, 1, True).cuda()
    dy = _rows((20000, 136), BF, 2).cuda()
    a = E.embedding_grad(dy, t, 900)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        b = E.embedding_grad(dy + 0, t + 0, 900)
    side.synchronize()
    assert torch.equal(a, b)


@CUDA
def test_refusals():
    from mamba3_b200 import embedding as E

    table = torch.zeros(10, 4, device="cuda")
    t = torch.zeros(3, dtype=torch.int64, device="cuda")
    dy = torch.zeros(3, 4, device="cuda")
    for bad in (lambda: E.embed_tokens(table[0], t), lambda: E.embed_tokens(table, t.float()),
                lambda: E.embed_tokens(table, t.cpu()), lambda: E.embed_tokens(table.double(), t),
                lambda: E.embed_tokens(table, t, dtype=torch.float16), lambda: E.embed_tokens(table.cpu(), t.cpu()),
                lambda: E.embedding_grad(dy, t[:2], 10), lambda: E.embedding_grad(dy, t, 0),
                lambda: E.embedding_grad(dy, t, 10, dtype=torch.float16),
                lambda: E.embedding_grad(dy, t, 10, out=torch.zeros(9, 4, device="cuda")),
                lambda: E.embedding_grad(dy, t, 10, out=torch.zeros(4, 10, device="cuda").t())):
        with pytest.raises(ValueError):
            bad()


def test_entry_points_check_their_arguments():
    from mamba3_b200 import _capi as C

    lib = C.lib()
    a = C.M3EmbedArgs()
    assert lib.m3_embed(None, None) == C.M3_ERR_ARG
    assert lib.m3_embed(a, None) == C.M3_ERR_SHAPE
    a.vocab, a.dim, a.rows_outer, a.rows_inner = 4, 8, 1, 0
    assert lib.m3_embed(a, None) == C.M3_OK  # nothing to do
    a.rows_inner = 2
    assert lib.m3_embed(a, None) == C.M3_ERR_ARG
    a.out_dtype = 3
    assert lib.m3_embed(a, None) == C.M3_ERR_UNSUPPORTED
    b = C.M3EmbedBwdArgs()
    assert lib.m3_embed_bwd(None, None) == C.M3_ERR_ARG
    assert lib.m3_embed_bwd(b, None) == C.M3_ERR_SHAPE
    b.vocab, b.dim, b.rows_outer, b.rows_inner, b.grad, b.tokens, b.dy, b.grad_ld = 4, 8, 1, 2, 256, 256, 256, 8
    assert lib.m3_embed_bwd(b, None) == C.M3_ERR_WORKSPACE
    need = lib.m3_embed_bwd_workspace_size(2, 8)
    assert need > 0 and lib.m3_embed_bwd_workspace_size(-1, 8) == 0
    b.workspace, b.workspace_bytes = 256, need - 1
    assert lib.m3_embed_bwd(b, None) == C.M3_ERR_WORKSPACE
    b.workspace, b.workspace_bytes = 264, need
    assert lib.m3_embed_bwd(b, None) == C.M3_ERR_WORKSPACE
