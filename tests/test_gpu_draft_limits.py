"""Draft verification where its numbers are at their ends."""
import numpy as np
import pytest

from sharplight_amd import native
from tests import step_ref
from tests.devutil import Dev, log
from tests.test_gpu_draft import Case
from tests.test_gpu_lora import held

pytestmark = pytest.mark.gpu


def _call(d, c, what, **kw):
    args, more = c.put(d, **kw)
    log(f"draft_verify {what}")
    native.draft_verify(*args, **more)
    native.synchronize()
    B = len(c.new)
    return d.get(c.at["out"], (B, c.stride), np.int32), d.get(c.at["n_out"], (B,), np.int32), d.get(c.at["logp"], (B, c.stride), np.float32)


# ---- random numbers at the ends ------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("drafts", ["none", "chosen", "chosen by a temperature"])
@pytest.mark.parametrize("low", [9.0, 4.0, 30.0])
def test_ends_beside_chunks_far_below(device, low, drafts, dtype):
    """The first and the last tokens lie `low` logits below the others at a temperature of 0.05 (2^-115 to 2^-866 of them), masked ones among
    and around them. Random numbers of 0 and 1 draw the first and the last token with a weight: none that is masked, none behind
    another that has a weight to speak of (2^-100 of the largest)."""
    V, wide = 30000, 8192  # the low ones fill the first and the last chunk of either type
    new = [1] * 6 if drafts == "none" else [2] * 6
    c = Case("ends", new, V, dtype, drafts == "chosen by a temperature", [0.05], [0.0], settle=False)
    z = c.rng.standard_normal((c.T, V)) * 0.1
    z[:, :wide] -= low
    z[:, -wide:] -= low
    z[c.rng.random((c.T, V)) < 0.5] = -np.inf
    z[:, :3], z[:, -3:] = -np.inf, -np.inf
    c.target, c.z = held(z, dtype)
    c.ids[:] = 15000  # a draft among the others, refused
    c.z[:, 15000] = 0.25
    c.target, c.z = held(c.z, dtype)
    c.accept[:] = 1 - 2.0 ** -24
    c.sample = np.float32([0.0, 1.0, 0.0, 2.0, np.nan, 1.0])
    with Dev() as d:
        out, n, logp = _call(d, c, f"ends low={low} {drafts} {dtype}")
    assert (n == 1).all()
    for i in range(6):
        p = step_ref.probabilities(c.z[c.starts[i]], 0.05)
        if drafts != "none":
            p[15000] = 0.0
        x = out[i, 0]
        assert p[x] >= 2.0 ** -150 * p.max(), (i, x, p[x], logp[i, 0])
        weighty = np.nonzero(p > 2.0 ** -100 * p.max())[0]
        if i in (0, 2, 4):
            assert x <= weighty[0]
        else:
            assert x >= weighty[-1]
