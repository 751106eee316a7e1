"""Refusals of the verification's C entry (no GPU)."""
import pytest

from cdq_lrr_b200 import _lib as L


@pytest.mark.parametrize("tokens,drafts", [
    (1 << 16, 1 << 16),                     # in place
    (1 << 16, (1 << 16) + 8 * 5 * 3 - 8),    # the drafts begin in the last token
    (1 << 16, (1 << 16) - 8 * 4 * 3 + 8),    # and end in the first
])
def test_tokens_over_drafts(tokens, drafts):
    """Three sequences of four drafts: the call reads drafts while others of its blocks write tokens."""
    f = L.lib().cdq_verify_drafts
    batch, k, vocab = 3, 4, 8
    need = batch * (k + 1) * L.VERIFY_ROW_BYTES
    assert f(4096, 40, 8, None, 0, 0, 0, drafts, 4096, 4096, batch, k, vocab, 1.0, tokens, None, 1 << 20, need, None) == 3
