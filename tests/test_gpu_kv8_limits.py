"""GPU tests of the paged 8-bit cache at the limits of what its calls take."""
import numpy as np
import pytest

from sharplight_amd import native
from tests import kv8_ref
from tests.devutil import Dev, log
from tests.test_gpu_kv8 import NP, Step, _advance, _attend, _cache, _check_advance, _check_write, _check_y, _from, _pattern, _put, _rng, _values

pytestmark = pytest.mark.gpu

# new, past, wide: a thread block a head; a shared line; row tiles; row tiles beside few rows
SHAPES = [([1, 1, 3], [0, 300, 65], 1), ([1, 1, 3], [0, 300, 65], 200), ([150], [90], 1), ([150, 20, 1], [0, 90, 333], 200)]


def _scores(c, st, q, G, scale):
    """The largest |z| that some row sees, before a cap."""
    top = 0.0
    for i, s in enumerate(st.slots):
        n = int(st.past[i]) + st.new[i]
        for h in range(c.heads):
            k = c.keys(st.pages[s, :-(-n // st.bs)], h)[0][:n]
            rows = q[st.starts[i]:st.starts[i + 1], h * G:(h + 1) * G].reshape(-1, c.D)
            top = max(top, float(np.abs(scale * (rows @ k.T)).max(initial=0)))
    return top


# ---- caps ------------------------------------------------------------------------------------------------------------

def _capped(fmt, dtype, cap, new, past, wide, D):
    """A cap far above the scores changes them by |z|^3 / (3 cap^2) at most, so y lies within the bound of uncapped attention and what
    the cap's arithmetic adds (below 1000, where it changes more, within the statement's bound, which grants 2^-22 of the cap). That is relative to z: the products by 1 / cap and by cap log2(e) and their factors, eight roundings
    of 2^-24, and 2^-21 for tanh (2^-22 of itself, of an argument off by 2^-22). A score that is off by d moves y by 2 d max|v| at most."""
    rng = _rng("caps", fmt, dtype, cap, len(new))
    heads, G, bs = 2, 2, 16
    st = Step(rng, new, past, bs, wide=wide)
    c = kv8_ref.Cache(fmt, st.blocks, bs, heads, D, fill=rng)
    q, q64 = _put(rng.standard_normal((st.T, heads * G, D)) * 3, dtype)
    scale = 0.125
    with Dev() as d:
        log(f"kv8_attention cap={cap} {dtype} {fmt} D={D} new={new} wide={wide}")
        y = _attend(d, dtype, st, c, q, G, scale=scale, softcap=cap)
        native.synchronize()
        got = _from(d.get(y, q.shape, NP[dtype]), dtype)
    cap = float(np.float32(cap))
    want, _ = kv8_ref.attention(c, q64, st.starts, st.past, st.slots, st.pages, scale=scale, softcap=cap, dtype=dtype)
    if cap < 1e3:
        _, bound = kv8_ref.attention(c, q64, st.starts, st.past, st.slots, st.pages, scale=scale, softcap=cap, dtype=dtype)
        return _check_y(got, want, bound, cap, _pattern(dtype))
    _, bound = kv8_ref.attention(c, q64, st.starts, st.past, st.slots, st.pages, scale=scale, dtype=dtype)
    z = _scores(c, st, q64, G, scale)
    most = kv8_ref.QMAX[fmt] * float(c.vs.max())
    _check_y(got, want, bound + 2 * most * ((8 * 2.0 ** -24 + 2.0 ** -21) * z + z ** 3 / (3 * cap * cap)), cap, _pattern(dtype))


@pytest.mark.parametrize("fmt,dtype", [("i8", "f32"), ("e4m3", "f32"), ("i8", "bf16"), ("e4m3", "bf16")])
@pytest.mark.parametrize("cap", [4e3, 1e5, 1e7, 1e9])
@pytest.mark.parametrize("new,past,wide", SHAPES)
def test_caps_above_the_scores(device, fmt, dtype, cap, new, past, wide):
    _capped(fmt, dtype, cap, new, past, wide, 64)


@pytest.mark.parametrize("cap", [255.0, 256.0, 257.0, 1e6])
@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("new,past,wide", SHAPES[1:3])
def test_caps_above_the_scores_of_wider_heads(device, cap, D, new, past, wide):
    _capped("i8", "bf16", cap, new, past, wide, D)


@pytest.mark.parametrize("fmt,dtype", [("i8", "f32"), ("e4m3", "bf16")])
@pytest.mark.parametrize("cap", [1e30, 1e38, 3.4e38])
@pytest.mark.parametrize("new,past,wide", SHAPES)
def test_caps_at_the_end_of_the_range(device, fmt, dtype, cap, new, past, wide):
    _capped(fmt, dtype, cap, new, past, wide, 64)


@pytest.mark.parametrize("fmt,dtype", [("i8", "f32"), ("e4m3", "bf16")])
@pytest.mark.parametrize("cap", [1e-6, 1.5e-38, 1e-39, 1e-45])
@pytest.mark.parametrize("new,past,wide", SHAPES)
def test_caps_near_zero(device, fmt, dtype, cap, new, past, wide):
    """Every score is about 0, that of a key of zeros among them: y is the mean of what a row sees. (The statement's bound counts the
    products before the cap too, so the capped scores' own error, at most the cap, is far inside it.)"""
    rng = _rng("tiny caps", fmt, dtype, cap, len(new))
    st = Step(rng, new, past, 16, wide=wide)
    c = kv8_ref.Cache(fmt, st.blocks, 16, 2, 64, fill=rng)
    c.k[:, :, 3::5] = 0
    q, q64 = _put(rng.standard_normal((st.T, 4, 64)) * np.exp2(rng.integers(0, 40, (st.T, 4, 1))), dtype)
    with Dev() as d:
        log(f"kv8_attention cap={cap} {dtype} {fmt} new={new} wide={wide}")
        y = _attend(d, dtype, st, c, q, 2, scale=0.125, softcap=cap)
        native.synchronize()
        got = _from(d.get(y, q.shape, NP[dtype]), dtype)
    cap = float(np.float32(cap))
    want, _ = kv8_ref.attention(c, q64, st.starts, st.past, st.slots, st.pages, scale=0.125, softcap=cap, dtype=dtype)
    _, bound = kv8_ref.attention(c, q64 * 2.0 ** -40, st.starts, st.past, st.slots, st.pages, scale=0.125, dtype=dtype)
    _check_y(got, want, bound + 4 * cap * kv8_ref.QMAX[fmt] * float(c.vs.max()), cap, _pattern(dtype))


# ---- scores and queries at the end of the range ------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kw", [dict(), dict(slopes=True), dict(window=200)])
@pytest.mark.parametrize("new,past,wide", [([1, 2], [130, 500], 1), ([1, 2], [130, 500], 200), ([40, 50], [130, 500], 1), ([60, 1], [130, 500], 200)])
def test_scores_far_below_zero(device, dtype, kw, new, past, wide):
    """Scores of -2^108 to -2^125, of which a row's highest is higher by a quarter, so its key's value is the answer. (The others' weights
    are 0: the rest is y's rounding and 2^-11 or 2^-22 of it for the weight, which cancels.)"""
    rng = _rng("far below", dtype, str(kw), len(new), new[0])
    st = Step(rng, new, past, 16, wide=wide)
    D, heads, G = 64, 2, 2
    c = kv8_ref.Cache("i8", st.blocks, 16, heads, D, fill=rng)
    c.k[:], c.ks[:], c.vs[:] = 0, 1.0, 1.0
    c.k[..., 0] = 256 - 120
    best = [p - 5 for p in past]  # every row of the request sees it, inside a window too
    for i, s in enumerate(st.slots):
        c.k[st.pages[s, best[i] // 16], :, best[i] % 16, 0] = 256 - 90
    q = np.zeros((st.T, heads * G, D))
    q[..., 0] = np.exp2(rng.integers(102, 118, (st.T, heads * G)))
    bits, _ = _put(q, dtype)
    with Dev() as d:
        log(f"kv8_attention scores far below zero {dtype} {kw} new={new} wide={wide}")
        slopes = d.put(np.full(heads * G, 0.25, np.float32)) if "slopes" in kw else None
        y = _attend(d, dtype, st, c, bits, G, scale=1.0, slopes=slopes, window=kw.get("window", 0))
        native.synchronize()
        got = _from(d.get(y, bits.shape, NP[dtype]), dtype)
    for i, s in enumerate(st.slots):
        v = c.v.view(np.int8)[st.pages[s, best[i] // 16], :, 0, :, best[i] % 16].astype(np.float64)  # [heads, D]
        rows = got[st.starts[i]:st.starts[i + 1]].reshape(-1, heads, G, D)
        assert (np.abs(rows - v[None, :, None]) <= np.abs(v[None, :, None]) * 2.0 ** (-20 if dtype == "f32" else -7)).all(), i


@pytest.mark.parametrize("fmt,dtype", [("i8", "f32"), ("e4m3", "bf16")])
@pytest.mark.parametrize("new,past,wide", [([1, 1, 3], [0, 300, 65], 1), ([1, 1, 3], [0, 300, 65], 200), ([150, 20, 1], [0, 90, 333], 200)])
def test_queries_that_are_not_finite(device, fmt, dtype, new, past, wide):
    """A row with an infinity or a NaN has no softmax: it is NaN, also where all its scores are -infinity, and no other row is. Under a cap
    an infinity counts as the cap."""
    rng = _rng("not finite", fmt, dtype, len(new), new[0])
    st = Step(rng, new, past, 16, wide=wide)
    c = kv8_ref.Cache(fmt, st.blocks, 16, 2, 64, fill=rng)
    one = 0x38 if fmt == "e4m3" else 1
    minus = 0xB8 if fmt == "e4m3" else 0xFF
    c.k[..., 0], c.k[..., 1], c.k[..., 2] = one, minus, np.where(rng.random(c.k.shape[:-1]) < 0.5, one, minus)
    x = rng.standard_normal((st.T, 4, 64)) * 3
    kind = rng.integers(0, 6, (st.T, 4))  # 0: -inf to all keys, 1: the same by a negative value, 2: either sign, 3: NaN, others finite
    kind[0] = [0, 1, 2, 4]
    x[kind == 0, 1], x[kind == 1, 0], x[kind == 2, 2], x[kind == 3, 9] = np.inf, -np.inf, np.inf, np.nan
    x[kind == 2, 5] = 1e30  # far beyond the others, and nothing beside an infinity
    q, q64 = _put(x, dtype)
    fine = np.where((kind > 3)[..., None], q64, 0.0)
    cap, scale = 4.0, 0.125
    for softcap in (0.0, cap):
        with Dev() as d:
            log(f"kv8_attention queries not finite {dtype} {fmt} new={new} wide={wide} cap={softcap}")
            y = _attend(d, dtype, st, c, q, 2, scale=scale, softcap=softcap)
            native.synchronize()
            got = _from(d.get(y, q.shape, NP[dtype]), dtype)
        want, bound = kv8_ref.attention(c, fine, st.starts, st.past, st.slots, st.pages, scale=scale, softcap=softcap, dtype=dtype)
        lost = kind <= 3 if softcap == 0 else kind == 3
        assert np.isnan(got[lost]).all(), np.argwhere(lost & ~np.isnan(got).all(-1))[:4].tolist()
        if softcap:  # the scores of an infinity: +-cap, as a query of that size along the one dim gives them without a cap
            sure = np.zeros(q64.shape)
            for k, dim, sign in ((0, 1, 1), (1, 0, -1), (2, 2, 1)):
                sure[kind == k, dim] = sign
            flat = c.copy()
            flat.ks[:] = 1.0
            w2, b2 = kv8_ref.attention(flat, sure, st.starts, st.past, st.slots, st.pages, scale=cap, dtype=dtype)
            turned = (kind <= 2)[..., None]
            want, bound = np.where(turned, w2, want), np.where(turned, b2 + 2 * 2.0 ** -22 * cap * kv8_ref.QMAX[fmt] * float(c.vs.max()), bound)
        _check_y(np.where(lost[..., None], want, got), want, bound, softcap)


# ---- requests and tables that do not fit ---------------------------------------------------------------------------------

@pytest.mark.parametrize("B", [3, 64, 70, 5000])
@pytest.mark.parametrize("bad", ["a row too many", "slot of no rows", "past of no rows"])
@pytest.mark.parametrize("new", [1, 40])
def test_write_reports_requests_without_rows_of_their_own(device, B, bad, new):
    """A request that begins behind the step's last row, and one that brings nothing but does not fit: reported like any other, and the
    others are written."""
    if new > 1 and B > 100:
        B = 130
    rng = _rng("reports", B, bad, new)
    counts, past = np.full(B, new), rng.integers(0, 40, B)
    at = B - 1 if bad == "a row too many" else int(rng.integers(0, B))
    counts[at] = 1 if bad == "a row too many" else 0
    st = Step(rng, counts.tolist(), past, 16)
    if bad == "a row too many":
        st.T -= 1
    elif bad == "slot of no rows":
        st.slots[at] = len(st.pages) + 5
    else:
        st.past[at] = st.pages.shape[1] * 16 + 1
    c = kv8_ref.Cache("i8", st.blocks, 16, 2, 32, fill=rng)
    k, k64 = _put(_values(rng, (st.T, 2, 32)), "f32")
    with Dev() as d:
        cache, where = _cache(d, c)
        log(f"kv8_write of {B} requests, {bad}")
        native.kv8_write("f32", d.put(k), d.put(k), cache, st.batch(d))
        with pytest.raises(native.SlhipCacheError, match=f"Request {at} .*does not fit"):
            native.synchronize()
        kv8_ref.write(c, k64, k64, st.starts, st.past, st.slots, st.pages)
        _check_write(d, c, where, bad)


@pytest.mark.parametrize("B,most", [(1, 100), (40, 100), (1030, 100), (30, 20000), (4096, 100)])
@pytest.mark.parametrize("bad", ["", "twice", "longer", "last"])
def test_release_of_blocks_that_are_not_held(device, B, most, bad):
    """A request that was released before, or with fewer blocks than its length says: nothing changes, and the next sync says why. Up to
    some 20000 blocks."""
    rng = _rng("held", B, bad, most)
    bs, bps = 16, -(-most // 16) + 2
    past = rng.integers(1, most, B).astype(np.int32)
    slots = rng.permutation(B + 2)[:B].astype(np.int32)
    pages, ids = np.full((B + 2, bps), -1, np.int32), iter(rng.permutation(B * bps).astype(np.int32))
    for s, p in zip(slots, past):
        for j in range(-(-int(p) // bs)):
            pages[s, j] = next(ids)
    at = B - 1 if bad == "last" else int(rng.integers(0, B))
    if bad == "twice":
        pages[slots[at]] = -1
    elif bad == "longer":  # ends within the row
        past[at] = -(-int(past[at]) // bs) * bs + 1
    elif bad == "last":
        pages[slots[at], -(-int(past[at]) // bs) - 1] = -1
    free = np.arange(9000, 9000 + B * bps + 9, dtype=np.int32)
    with Dev() as d:
        where = {"pages": d.put(pages), "free": d.put(free), "n": d.put(np.int32([5])), "out": d.put(np.int32([77]))}
        p = native.kv_pages(B, d.put(past), None, where["pages"], pages.shape[0], bps, bs, where["free"], len(free), where["n"], where["out"],
                            slots=d.put(slots))
        log(f"kv_pages_release of {B} requests, {bad}")
        native.kv_pages_release(p)
        n_free = 5
        if bad:
            with pytest.raises(native.SlhipCacheError, match=f"request {at} .*does not hold"):
                native.synchronize()
        else:
            native.synchronize()
            ok, pages, free, n_free = kv8_ref.release(past, slots, pages, bs, free, 5)
            assert ok
        assert np.array_equal(d.get(where["pages"], pages.shape, np.int32), pages)
        assert np.array_equal(d.get(where["free"], free.shape, np.int32), free)
        assert d.get(where["out"], (1,), np.int32)[0] == n_free


@pytest.mark.parametrize("tokens", [(1 << 31) - 1, (1 << 31) - 2])
def test_advance_of_more_tokens_than_any_step_has(device, tokens):
    """Two requests of neighbouring places whose tokens together pass 2^31, in a step without rows: refused."""
    B, bs, bps = 1500, 1 << 20, 1600
    past, count, slot = np.zeros(B, np.int32), np.zeros(B, np.int32), np.arange(B, dtype=np.int32)
    count[:2] = 1600 << 20
    pages, free = np.full((B, bps), -1, np.int32), np.arange(4000, dtype=np.int32)
    with Dev() as d:
        p, at = _advance(d, past, count, slot, pages, bs, free, len(free), 1, False, rows=False)
        p.tokens = tokens
        log(f"kv_pages_advance of {2 * int(count[0])} tokens")
        native.kv_pages_advance(p)
        with pytest.raises(native.SlhipCacheError, match="more tokens than rows"):
            native.synchronize()
        _check_advance(d, at, (False, pages, len(free), np.zeros(B + 1, np.int32), None, None), B, 0, rows=False)


# ---- workspace -------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("f32", 64), ("bf16", 256)])
def test_one_workspace_for_every_smaller_step(device, dtype, D):
    """A workspace of the size that the largest batch asks for takes all smaller steps: fewer requests, rows and new tokens, shorter tables."""
    heads, G, bs = 2, 4, 16
    steps = [([700, 600, 500, 40], [2500, 0, 900, 5], 150, 0), ([300], [2000], 150, 0), ([128], [3300], 0, 128), ([20, 9], [3000, 100], 20, 0),
             ([4, 1, 3], [3000, 100, 2600], 0, 4), ([8], [1500], 0, 8), ([1], [100], 150, 1), ([40], [600], 0, 0)]
    with Dev() as d:
        sizes = []
        for k, (new, past, wide, max_new) in enumerate(steps):
            rng = _rng("workspace", dtype, D, k)
            st = Step(rng, new, past, bs, wide=wide)
            c = kv8_ref.Cache("i8", st.blocks, bs, heads, D, fill=rng)
            q, q64 = _put(rng.standard_normal((st.T, heads * G, D)) * 2, dtype)
            cache, batch = _cache(d, c)[0], st.batch(d)
            if k == 0:  # the table's rows as long as any, and more rows than the step has
                largest = native.kv8_batch(4, 9000, *st.dev[:3], 8, 360)
                need = native.kv8_attention_work_bytes(heads * G, cache, largest, 0)
                work = d.empty(need, fill=0xFF)
            sizes.append(native.kv8_attention_work_bytes(heads * G, cache, batch, max_new))
            y = d.empty(q.nbytes, fill=0x5A)
            log(f"kv8_attention {dtype} D={D} new={new} past={past} of a workspace of {need} bytes")
            native.kv8_attention(dtype, d.put(q), y, heads * G, cache, batch, scale=0.125, max_new=max_new, work=work, work_bytes=need)
            native.synchronize()
            want, bound = kv8_ref.attention(c, q64, st.starts, st.past, st.slots, st.pages, scale=0.125, dtype=dtype)
            _check_y(_from(d.get(y, q.shape, NP[dtype]), dtype), want, bound, new, _pattern(dtype))
        assert max(sizes) <= need
