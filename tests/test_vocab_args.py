"""What the vocabulary-end operators refuse before anything is launched (no GPU needed)."""

import torch

from mamba3_b200 import _capi as C
from mamba3_b200 import _tensors as T


def test_scoring_refuses_more_rows_than_its_indices_hold():
    a = C.M3ScoreArgs()
    a.vocab, a.temperature, a.logits, a.entropy, a.lse = 10, 1.0, 16, 16, 16
    # 2^32 + 65536 rows would be cut to 65536, 2^31 to a negative count, 2^30 + 1024 passes 2^30
    for outer, inner in ((65536, 65537), (65536, 32768), (1 << 20, 1025)):
        a.rows_outer, a.rows_inner = outer, inner
        assert C.lib().m3_token_logprobs(a, None) == C.M3_ERR_SHAPE
    a.rows_outer, a.rows_inner = -1, 4
    assert C.lib().m3_token_logprobs(a, None) == C.M3_ERR_SHAPE
    a.rows_outer = 0
    assert C.lib().m3_token_logprobs(a, None) == C.M3_OK


def test_memory_apart():
    """Every pair of views of one buffer: certain to be apart only if no byte is in both, and found to be where
    the views are column ranges of one pitch."""
    buf = torch.zeros(6, 24)
    flat = buf.view(-1)
    views = [buf[:, lo:lo + w] for lo in (0, 3, 8, 16) for w in (1, 5, 8)]
    views += [flat[lo:lo + 40].view(5, 8) for lo in (0, 20, 41, 80)] + [flat[24:48], buf[2], buf[::2, 8:16], buf[:0]]
    views += [buf.view(torch.bfloat16)[:, lo:lo + 8] for lo in (0, 6, 16, 40)] + [buf.view(3, 2, 24)[:, :, 4:6]]

    def held(t):
        at = torch.zeros(6 * 24 * 4, dtype=torch.bool)
        idx = torch.arange(6 * 24 * 4 // t.element_size()).as_strided(t.shape, t.stride(), t.storage_offset())
        for i in idx.reshape(-1).tolist():
            at[i * t.element_size():(i + 1) * t.element_size()] = True
        return at

    for a in views:
        for b in views:
            meet = bool((held(a) & held(b)).any())
            assert not (meet and T.apart(a, b))
            if a.dim() == b.dim() == 2 and a.stride(0) == b.stride(0) == 24:
                assert T.apart(a, b) == (not meet)


def test_distillation_refuses_temperatures_whose_square_is_no_number():
    a = C.M3DistillArgs()
    a.rows_outer, a.rows_inner, a.vocab, a.k = 1, 1, 10, 3
    a.logits, a.ids, a.teacher, a.row_loss = 16, 16, 16, 16
    for t in (1e19, 1e30):
        a.temperature = t
        assert C.lib().m3_distill(a, None) == C.M3_ERR_ARG


def test_embedding_gradient_refuses_widths_before_it_writes():
    """The widest rows that the launches' grids reach: 65535 times 8 threads' columns, 1, 2 or 8 a thread."""
    a = C.M3EmbedBwdArgs()
    a.rows_outer, a.rows_inner, a.vocab, a.scale = 1, 1000, 4, 1.0  # more than one chunk of rows
    a.tokens, a.grad, a.workspace, a.workspace_bytes = 16, 256, 256, 1 << 40
    for dim, dy in ((65535 * 8 + 1, 256), (65535 * 16 + 2, 256), (65535 * 64 + 8, 256), (65535 * 8 + 8, 260)):
        a.dim = a.grad_ld = a.dy_inner = a.dy_outer = dim
        a.dy = dy
        assert C.lib().m3_embed_bwd(a, None) == C.M3_ERR_SHAPE
