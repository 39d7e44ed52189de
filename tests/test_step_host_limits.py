"""Host-side checks of draft verification at the limits of its sizes."""
import pytest

from sharplight_amd import native
from tests.test_kv8_host import FAKE
from tests.test_step_host import _drafts

HUGE = [(1, 1 << 62, 16384), (1, 1 << 61, 8 * 4096), (1, 1 << 60, 1 << 16), (1, (1 << 63) - 1, 1 << 24), (1, 1, (1 << 63) - 1), (1 << 62, 1, 16384)]


@pytest.mark.parametrize("requests,tokens,vocab", HUGE)
def test_sizes_whose_products_pass_64_bits_are_refused(requests, tokens, vocab):
    """2^62 rows of four chunks are 2^64 chunks, which is 0 in 64 bits: no workspace of a few bytes is enough for them."""
    assert native.draft_verify_work_bytes(requests, tokens, vocab) == -1
    with pytest.raises(NotImplementedError, match="too many"):
        native.draft_verify("f32", FAKE, FAKE, _drafts(requests=requests, tokens=tokens, vocab=vocab), work=FAKE, work_bytes=1 << 40)
