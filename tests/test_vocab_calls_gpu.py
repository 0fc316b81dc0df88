"""The vocabulary-end operators as torch calls: what autograd is told of writes, and what is refused."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _lists(rows, vocab, k=5, seed=0):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, vocab, (rows, k), generator=g).cuda()
    return torch.randn(rows, vocab, generator=g).cuda(), ids, torch.randn(rows, k, generator=g).cuda()


@pytest.mark.parametrize("vocab", [300, 9000])
def test_overwritten_logits_are_not_differentiated(vocab):
    """Another loss saved the logits that ``out=`` then overwrites: its backward must not run on the gradient."""
    from mamba3_b200 import distill as D

    x, ids, teacher = _lists(6, vocab)
    leaf = x.clone().requires_grad_(True)
    for other in (lambda t: torch.logsumexp(t, -1).square().sum(), lambda t: D.distill_loss(t, ids, teacher)):
        logits = leaf * 1.0
        loss, view = other(logits), logits.detach()
        before = logits._version
        D.distill_loss_and_grad(view, ids, teacher, out=view)
        assert logits._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    # memory of its own: the other loss goes on
    logits = leaf * 1.0
    loss = torch.logsumexp(logits, -1).square().sum()
    D.distill_loss_and_grad(logits.detach(), ids, teacher, out=torch.empty_like(x))
    loss.backward()
    with torch.inference_mode():  # tensors without a version
        y = x.clone()
        _, dx = D.distill_loss_and_grad(y, ids, teacher, out=y)
    assert torch.equal(dx, D.distill_loss_and_grad(x, ids, teacher)[1])


def test_table_added_to_is_not_differentiated():
    from mamba3_b200 import embedding as E

    leaf = torch.randn(20, 8, device="cuda").requires_grad_(True)
    held = leaf * 1.0
    loss = held.square().sum()
    tokens, dy = torch.arange(5, device="cuda"), torch.ones(5, 8, device="cuda")
    E.embedding_grad(dy, tokens, 20, out=held.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_gradient_is_not_added_to_the_memory_it_is_read_from():
    from mamba3_b200 import embedding as E

    tokens = torch.tensor([1, 0, 1, 3], device="cuda")
    buf = torch.ones(4, 24, device="cuda")
    flat = buf.view(-1)
    for dy, out in ((buf[:, :8], buf[:, :8]), (buf[:, :8], buf[:, 4:12]), (flat[:32].view(4, 8), flat[16:48].view(4, 8)),
                    (flat[:32].view(4, 8), buf[:, :8]),
                    (buf.view(torch.bfloat16)[:, 8:16], buf[:, :8])):  # half the bytes an element
        with pytest.raises(ValueError, match="share no memory"):
            E.embedding_grad(dy, tokens, 4, out=out)
    assert (buf == 1).all()
    # columns of one buffer that do not meet, and memory apart
    E.embedding_grad(buf[:, :8], tokens, 4, out=buf[:, 8:16])
    want = torch.tensor([2.0, 3.0, 1.0, 2.0], device="cuda")[:, None].expand(4, 8)
    assert torch.equal(buf[:, 8:16], want) and (buf[:, :8] == 1).all() and (buf[:, 16:] == 1).all()
    E.embedding_grad(flat[:32].view(4, 8), tokens, 4, out=flat[64:96].view(4, 8))


def test_gradient_is_not_added_to_a_leaf():
    from mamba3_b200 import embedding as E

    tokens, dy = torch.arange(3, device="cuda"), torch.ones(3, 8, device="cuda")
    leaf = torch.zeros(4, 8, device="cuda").requires_grad_(True)
    with pytest.raises(ValueError, match="leaf"):
        E.embedding_grad(dy, tokens, 4, out=leaf)
    assert not leaf.any()
    with torch.no_grad():  # as torch's own in-place operations
        E.embedding_grad(dy, tokens, 4, out=leaf)
    assert (leaf[:3] == 1).all() and not leaf[3].any()


def test_forward_mode_is_refused():
    """There is no forward-mode derivative; a result without its tangent would be a derivative of 0."""
    import torch.autograd.forward_ad as fw
    from mamba3_b200 import distill as D
    from mamba3_b200 import embedding as E

    x, ids, teacher = _lists(4, 50)
    tokens = ids[:, 0]
    with fw.dual_level():
        dual = fw.make_dual(x, torch.ones_like(x))
        for mode in (torch.enable_grad(), torch.no_grad()):
            with mode:
                for reduction in ("mean", "sum", "none"):
                    with pytest.raises(NotImplementedError):
                        D.distill_loss(dual, ids, teacher, reduction=reduction)
                with pytest.raises(NotImplementedError):
                    E.embed_tokens(dual, tokens % 4)
                D.distill_loss(x, ids, teacher)  # tensors without a tangent go on
                E.embed_tokens(x, tokens % 4)


def test_a_failed_call_does_not_fail_the_next():
    """Rows too wide for the gradient's launches are refused; the call after it is not blamed for that."""
    from mamba3_b200 import embedding as E

    dim = 600001  # odd: one column a thread
    tokens, dy = torch.arange(40, device="cuda") % 4, torch.ones(40, dim, device="cuda")
    with pytest.raises(ValueError):
        E.embedding_grad(dy, tokens, 4)
    out = E.embed_tokens(torch.ones(4, 8, device="cuda"), tokens, scale=3.0)
    assert (out == 3).all()


def test_sizes_past_32_bits_are_refused():
    """A vocabulary of 2^32 + 256 is not one of 256."""
    from mamba3_b200 import distill as D
    from mamba3_b200 import embedding as E
    from mamba3_b200 import scoring as S

    one = torch.zeros(1, dtype=torch.bfloat16, device="cuda")
    logits = one.expand(2 ** 32 + 256)  # no memory of that size
    ids, teacher = torch.zeros(3, dtype=torch.int64, device="cuda"), torch.zeros(3, device="cuda")
    for call in (lambda: S.token_logprobs(logits), lambda: D.distill_loss(logits, ids, teacher),
                 lambda: D.distill_loss_and_grad(logits, ids, teacher),
                 lambda: E.embed_tokens(one[:, None].expand(2 ** 32 + 8, 1), ids),
                 lambda: E.embedding_grad(torch.zeros(3, 1, device="cuda"), ids, 2 ** 32 + 8)):
        with pytest.raises(ValueError, match="vocab"):
            call()
