"""What a step back leaves in the 8-bit cache (slhip_kv_pages_trim behind slhip_kv8_write): the codes and scales of blocks that are kept."""
import numpy as np
import pytest

from sharplight_amd import native
from tests import kv8_ref
from tests.devutil import Dev, log
from tests.test_gpu_kv8 import _check_write
from tests.test_gpu_lora import held, rng_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("refused", [300.0, np.inf, np.nan])
def test_blocks_that_keep_some_of_their_tokens(device, fmt, refused):
    """Two requests cache 20 tokens, then check drafts whose values are `refused` and step back to 20 and to 16: the first one's second block
    keeps its tokens under the scale (or the NaN) that the drafts gave it, the second one's went back and is begun anew. Writing a block's tokens again
    from its first one on undoes it."""
    rng = rng_of("keep", fmt, refused)
    B, bs, bps, blocks, heads, D = 2, 16, 4, 10, 2, 32
    c = kv8_ref.Cache(fmt, blocks, bs, heads, D, fill=rng)
    at = {k: np.int32(v) for k, v in (("slots", [1, 0]), ("free", rng.permutation(blocks)), ("n", [blocks]))}
    with Dev() as d:
        codes = [d.put(x) for x in (c.k, c.v, c.ks, c.vs)]
        cache = native.kv8_cache(fmt, *codes, blocks, bs, heads, D)
        p = {k: d.put(v) for k, v in at.items()} | {k: d.empty(4 * n) for k, n in (("past", B), ("count", B), ("starts", B + 1))}
        p["pages"] = d.put(np.full((B, bps), -1, np.int32))
        pk, pv = d.empty(4 * 64 * heads * D), d.empty(4 * 64 * heads * D)

        def tables(past, count, T):
            for k, v in (("past", past), ("count", count)):
                v = np.int32(v)
                native.call("slhip_memcpy_h2d", p[k], v.ctypes.data, v.nbytes, None)
            return native.kv_pages(B, p["past"], p["count"], p["pages"], B, bps, bs, p["free"], blocks, p["n"], p["n"], T, p["starts"], slots=p["slots"])

        def step(what, past, count, make, advance=True):
            T = sum(count)
            k, v = (held(make(rng.standard_normal((T, heads, D))), "f32") for _ in range(2))
            t = tables(past, count, T)
            log(f"{what} {fmt} {refused}")
            if advance:
                native.kv_pages_advance(t)
            else:
                starts = np.int32([0, *np.cumsum(count)])
                native.call("slhip_memcpy_h2d", p["starts"], starts.ctypes.data, starts.nbytes, None)
            for to, x in ((pk, k[0]), (pv, v[0])):
                native.call("slhip_memcpy_h2d", to, x.ctypes.data, x.nbytes, None)
            native.kv8_write("f32", pk, pv, cache, native.kv8_batch(B, T, p["starts"], p["past"], p["pages"], B, bps, slots=p["slots"]))
            native.synchronize()
            pages = d.get(p["pages"], (B, bps), np.int32)
            kv8_ref.write(c, k[1], v[1], np.concatenate([[0], np.cumsum(count)]), past, at["slots"], pages)
            _check_write(d, c, codes, what)
            return pages

        step("prompt", [0, 0], [20, 20], lambda x: x)
        # one draft's value is refused's in both requests
        pages = step("drafts", [20, 20], [3, 3], lambda x: np.where((np.arange(6) % 3 == 1)[:, None, None], refused, x))
        native.kv_pages_trim(tables([20, 16], [3, 7], 0))
        native.synchronize()
        _check_write(d, c, codes, "trim")
        mixed, gone = pages[at["slots"][0], 1], pages[at["slots"][1], 1]
        assert d.get(p["pages"], (B, bps), np.int32)[at["slots"][1], 1] == -1
        grown = c.ks[mixed].copy()
        pages = step("next tokens", [20, 16], [1, 1], lambda x: x)
        assert pages[at["slots"][1], 1] == gone  # taken again, and begun anew
        assert np.isnan(grown).all() == (not np.isfinite(refused))
        assert np.array_equal(c.ks[mixed], grown, equal_nan=True) and (c.ks[gone] < 1).all()
        step("again from the block's first token", [16, 17], [5, 1], lambda x: x, advance=False)
        assert (c.ks[mixed] < 1).all()
