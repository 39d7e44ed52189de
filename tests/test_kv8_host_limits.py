"""Host-side checks of the paged 8-bit cache at the limits of its calls."""
import numpy as np
import pytest

from sharplight_amd import native
from tests.test_kv8_host import FAKE, _batch, _cache


@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("heads,q_heads", [(1, 1), (8, 32), (2, 34), (2, 128), (4, 4), (512, 512)])
def test_a_workspace_takes_every_smaller_step(head_dim, heads, q_heads):
    """No step of fewer requests, rows, new tokens or shorter table rows needs more than the largest does."""
    cache = _cache(heads=heads, head_dim=head_dim)
    need = lambda b, t, w, m: native.kv8_attention_work_bytes(q_heads, cache, _batch(requests=b, tokens=t, blocks_per_slot=w, page_slots=4096), m)  # noqa: E731
    rng = np.random.default_rng(head_dim * 1000 + q_heads)
    log = lambda top: int(np.exp2(rng.uniform(0, np.log2(top + 1))))  # noqa: E731
    for _ in range(300):
        b, t, w, m = max(log(2000), 1), max(log(20000), 1), max(log(40000), 1), log(300)
        most = need(b, t, w, m)
        assert 0 <= most < 1 << 28
        for _ in range(30):
            b2, t2, w2 = 1 + int(rng.integers(0, b)), 1 + log(t) % t, 1 + log(w) % w
            # of a step with a limit, new tokens within it; a step without one has its rows as the limit
            m2 = 1 + log(m) % m if m else int(rng.integers(0, 2)) * (1 + log(t2) % t2)
            got = need(b2, t2, w2, m2)
            assert got <= most, ((b, t, w, m), (b2, t2, w2, m2), got, most)


def test_a_prompt_and_its_last_chunk():
    """A long prompt fills the machine without a workspace; the shorter step after it does not."""
    need = lambda t: native.kv8_attention_work_bytes(32, _cache(heads=8, head_dim=128), _batch(requests=1, tokens=t, blocks_per_slot=512), 0)  # noqa: E731
    assert need(8192) >= need(1024) >= need(128) > 0


def test_launches_of_wide_heads_past_their_limits_are_refused():
    """Row tiles of 256 dims have 512 threads: 2^23 of them are a launch of 2^32."""
    for tokens in (300 << 20, 500 << 20):
        with pytest.raises(NotImplementedError, match="too many tiles"):
            native.kv8_attention("bf16", FAKE, FAKE, 4, _cache(head_dim=256), _batch(tokens=tokens, blocks_per_slot=1000), scale=1.0,
                                 work=FAKE, work_bytes=1 << 40)
