"""What the C entries of the vocabulary-end operators refuse before anything is launched (no GPU needed)."""

from mamba3_b200 import _capi as C


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
