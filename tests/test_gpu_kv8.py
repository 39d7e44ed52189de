"""GPU parity of the paged 8-bit cache: its block tables (whole numbers: equal), its write (codes and scales: bit for bit)
and its attention, against the 64-bit statements of tests/kv8_ref.py; for the attention within the bound derived there."""
import zlib

import numpy as np
import pytest

import oracle
from sharplight_amd import native
from tests import kv8_ref
from tests.devutil import Dev, log

pytestmark = pytest.mark.gpu


def _rng(*parts):
    return np.random.default_rng(zlib.crc32(repr(parts).encode()))


def _put(x, dtype):
    """f64 values as an array of the dtype, and the values it then holds."""
    f = x.astype(np.float32)
    if dtype == "f32":
        return f, f.astype(np.float64)
    b = oracle.to_bf16(f)
    return b, oracle.from_bf16(b).astype(np.float64)


def _from(bits, dtype):
    return (bits if dtype == "f32" else oracle.from_bf16(bits)).astype(np.float64)


NP = {"f32": np.float32, "bf16": np.uint16}


class Step:
    """A step's requests with block tables that scatter their blocks over a cache of a few blocks more."""

    def __init__(self, rng, new, past, bs, spare=3, padding=0, wide=1):
        self.new, self.past, self.bs = list(new), np.int32(past), bs
        B = len(self.new)
        need = [-(-(a + b) // bs) for a, b in zip(new, past)]
        ids = rng.permutation(sum(need) + spare).astype(np.int32)
        self.blocks = len(ids)
        self.slots = rng.permutation(B + 2)[:B].astype(np.int32)
        self.pages = np.full((B + 2, max(need + [1]) + wide), -1, np.int32)
        at = 0
        for s, n in zip(self.slots, need):
            self.pages[s, :n] = ids[at:at + n]
            at += n
        self.starts = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)
        self.T = int(self.starts[-1]) + padding

    def batch(self, d):
        self.dev = [d.put(x) for x in (self.starts, self.past, self.pages, self.slots)]
        return native.kv8_batch(len(self.new), self.T, self.dev[0], self.dev[1], self.dev[2], self.pages.shape[0],
                                self.pages.shape[1], slots=self.dev[3])


def _cache(d, c):
    at = [d.put(x) for x in (c.k, c.v, c.ks, c.vs)]
    return native.kv8_cache(c.fmt, *at, c.blocks, c.bs, c.heads, c.D), at


def _get_cache(d, c, at):
    return [d.get(p, x.shape, x.dtype) for p, x in zip(at, (c.k, c.v, c.ks, c.vs))]


# ---- block tables --------------------------------------------------------------------------------------------------

def _tables(rng, B, bs, most_past, most_new, slots, spare=5):
    past = rng.integers(0, most_past + 1, B).astype(np.int32)
    count = rng.integers(0, most_new + 1, B).astype(np.int32)
    past[: B // 3] -= past[: B // 3] % bs  # some at a block's border
    bps = -(-(most_past + most_new) // bs)
    slot = rng.permutation(slots)[:B].astype(np.int32)
    pages = np.full((slots, bps), -1, np.int32)
    ids = iter(rng.permutation(B * bps + 100).astype(np.int32))
    for i in range(B):
        for j in range(-(-int(past[i]) // bs)):
            pages[slot[i], j] = next(ids)
    need = sum(-(-(int(p) + int(c)) // bs) - -(-int(p) // bs) for p, c in zip(past, count))
    free = np.int32([next(ids) for _ in range(min(need + spare, 100 + need))])
    return past, count, slot, pages, free, need


def _advance(d, past, count, slot, pages, bs, free, n_free, tokens, in_place, with_slots=True, rows=True, shift=0):
    B = len(past)
    at = {"pages": d.put(pages), "free": d.put(free) if len(free) else d.empty(4), "n": d.put(np.int32([n_free])), "out": d.put(np.int32([77])),
          "starts": d.empty(4 * (B + 1)), "seq": d.empty(16 * tokens, pad_bytes=shift), "pos": d.empty(4 * tokens)}
    if in_place:
        at["out"] = at["n"]
    p = native.kv_pages(B, d.put(past), d.put(count), at["pages"], pages.shape[0], pages.shape[1], bs, at["free"], len(free),
                        at["n"], at["out"], tokens, at["starts"], seq=at["seq"] if rows else None,
                        pos=at["pos"] if rows else None, slots=d.put(slot) if with_slots else None)
    return p, at


def _check_advance(d, at, want, B, tokens, rows=True):
    ok, pages, n_free, starts, seq, pos = want
    assert np.array_equal(d.get(at["pages"], pages.shape, np.int32), pages)
    assert d.get(at["out"], (1,), np.int32)[0] == n_free
    assert np.array_equal(d.get(at["starts"], (B + 1,), np.int32), starts)
    if rows and tokens:
        assert np.array_equal(d.get(at["seq"], (tokens, 4), np.int32), seq)
        assert np.array_equal(d.get(at["pos"], (tokens,), np.int32), pos)


@pytest.mark.parametrize("B,bs,most_past,most_new,padding,in_place", [
    (1, 16, 0, 1, 0, True), (1, 16, 40, 40, 7, False), (3, 1, 5, 3, 2, True), (64, 16, 500, 1, 0, True), (65, 32, 300, 40, 3, False),
    (333, 64, 1000, 30, 1, True), (1100, 16, 50, 2, 9, False), (4096, 16, 33, 1, 0, True), (7, 16, 100, 1500, 0, True),
    (40, 128, 3000, 400, 11, False), (5, 16, 20, 0, 4, True)])
def test_pages_advance(device, B, bs, most_past, most_new, padding, in_place):
    rng = _rng("advance", B, bs, most_past, most_new)
    past, count, slot, pages, free, need = _tables(rng, B, bs, most_past, most_new, B + 3)
    tokens = int(count.sum()) + padding
    n_free = len(free) - 2 if len(free) > need + 2 else len(free)
    with Dev() as d:
        log(f"kv_pages_advance B={B} bs={bs} tokens={tokens}")
        p, at = _advance(d, past, count, slot, pages, bs, free, n_free, tokens, in_place, shift=4 if B % 2 else 0)
        native.kv_pages_advance(p)
        native.synchronize()
        want = kv8_ref.advance(past, count, slot, pages, bs, free, n_free, tokens)
        assert want[0]
        _check_advance(d, at, want, B, tokens)
        assert np.array_equal(d.get(at["free"], free.shape, np.int32), free)


def test_pages_of_the_largest_table(device):
    """4096 requests in a table of 131072 rows, the last row among them, and rows over hundreds of thread blocks."""
    rng = _rng("largest")
    B, bs, slots = 4096, 64, 131072
    past = rng.integers(0, 128, B).astype(np.int32)
    count = np.where(rng.random(B) < 0.1, rng.integers(0, 129, B), 1).astype(np.int32)
    slot = rng.permutation(slots)[:B].astype(np.int32)
    slot[7] = slots - 1 if (slot != slots - 1).all() else slot[7]
    pages = np.full((slots, 4), -1, np.int32)
    for i in range(B):
        n = -(-int(past[i]) // bs)
        pages[slot[i], :n] = 10 * i + np.arange(n)
    need = int(sum(-(-(int(p) + int(c)) // bs) - -(-int(p) // bs) for p, c in zip(past, count)))
    free, tokens = (100000 + rng.permutation(need + 9)).astype(np.int32), int(count.sum()) + 100
    for in_place in (False, True):
        with Dev() as d:
            log(f"kv_pages_advance of {B} requests, {tokens} rows, in place: {in_place}")
            p, at = _advance(d, past, count, slot, pages, bs, free, len(free), tokens, in_place)
            native.kv_pages_advance(p)
            native.synchronize()
            _check_advance(d, at, kv8_ref.advance(past, count, slot, pages, bs, free, len(free), tokens), B, tokens)


def test_pages_identity_slots_no_rows_and_no_requests(device):
    rng = _rng("identity")
    past, count, slot, pages, free, need = _tables(rng, 9, 16, 60, 20, 9)
    order = np.argsort(slot)
    past, count, slot = past[order], count[order], slot[order]
    with Dev() as d:
        p, at = _advance(d, past, count, slot, pages, 16, free, len(free), int(count.sum()), False, with_slots=False, rows=False)
        log("kv_pages_advance without slots and rows")
        native.kv_pages_advance(p)
        native.synchronize()
        _check_advance(d, at, kv8_ref.advance(past, count, slot, pages, 16, free, len(free), int(count.sum())), 9, 0, rows=False)
        p, at = _advance(d, past[:0], count[:0], slot[:0], pages, 16, free, len(free), 6, False)
        log("kv_pages_advance of no requests")
        native.kv_pages_advance(p)
        native.synchronize()
        _check_advance(d, at, kv8_ref.advance([], [], [], pages, 16, free, len(free), 6), 0, 6)


@pytest.mark.parametrize("case", ["free", "rows", "slot", "negative_slot", "twice", "length", "past", "count", "n_free"])
@pytest.mark.parametrize("many", [False, True])
def test_pages_that_do_not_fit(device, case, many):
    """Nothing changes but starts and rows (all padding), and the next sync says why."""
    rng = _rng("bad", case)
    B = 70
    past, count, slot, pages, free, need = _tables(rng, B, 16, 200, 90 if many else 8, B + 3, spare=0)
    count[-1] = 20
    need = sum(-(-(int(p) + int(c)) // 16) - -(-int(p) // 16) for p, c in zip(past, count))
    free = np.arange(1000, 1000 + need, dtype=np.int32)
    tokens, n_free = int(count.sum()), len(free)
    if case == "free":
        n_free -= 1
    elif case == "rows":
        tokens -= 1
    elif case == "slot":
        slot[40] = B + 3
    elif case == "negative_slot":
        slot[40] = -1
    elif case == "twice":
        slot[40] = slot[41]
    elif case == "length":
        past[40] = pages.shape[1] * 16 - int(count[40]) + 1
    elif case == "past":
        past[40] = -1
    elif case == "count":
        count[40] = -1
    elif case == "n_free":
        n_free += 1
    with Dev() as d:
        log(f"kv_pages_advance that does not fit: {case}")
        p, at = _advance(d, past, count, slot, pages, 16, free, n_free, tokens, False)
        native.kv_pages_advance(p)
        why = {"free": "free list", "n_free": "free list", "rows": "more tokens than rows"}.get(case, "slot is outside" if case in ("slot", "negative_slot", "twice") else "lengths")
        with pytest.raises(native.SlhipCacheError, match=why):
            native.synchronize()
        want = kv8_ref.advance(past, count, slot, pages, 16, free, n_free, tokens)
        assert not want[0]
        _check_advance(d, at, want, B, tokens)


@pytest.mark.parametrize("B,bs", [(1, 16), (33, 16), (1030, 32)])
@pytest.mark.parametrize("short", [False, True])
def test_pages_release(device, B, bs, short):
    rng = _rng("release", B, bs)
    past, count, slot, pages, free, need = _tables(rng, B, bs, 400, 1, B + 3)
    held = sum(-(-int(p) // bs) for p in past)
    past[0] = max(past[0], 1) if pages[slot[0], 0] >= 0 else past[0]
    n_free = 4
    free = np.arange(5000, 5000 + n_free + held + 3 - (4 if short and held else 0), dtype=np.int32)
    if short and not held:
        pytest.skip("nothing to release")
    with Dev() as d:
        at = {"pages": d.put(pages), "free": d.put(free), "n": d.put(np.int32([n_free]))}
        p = native.kv_pages(B, d.put(past), None, at["pages"], pages.shape[0], pages.shape[1], bs, at["free"], len(free), at["n"], at["n"],
                            slots=d.put(slot))
        log(f"kv_pages_release B={B} short={short}")
        native.kv_pages_release(p)
        ok, wp, wf, wn = kv8_ref.release(past, slot, pages, bs, free, n_free)
        assert ok != short
        if short:
            with pytest.raises(native.SlhipCacheError, match="free list"):
                native.synchronize()
        native.synchronize()
        assert np.array_equal(d.get(at["pages"], wp.shape, np.int32), wp)
        assert np.array_equal(d.get(at["free"], wf.shape, np.int32), wf)
        assert d.get(at["n"], (1,), np.int32)[0] == wn


# ---- write -----------------------------------------------------------------------------------------------------------

def _check_write(d, c, at, what):
    for name, got, want in zip(("k codes", "v codes", "k scales", "v scales"), _get_cache(d, c, at), (c.k, c.v, c.ks, c.vs)):
        same = (got == want) if got.dtype == np.uint8 else (got.view(np.uint32) == want.view(np.uint32)) | (np.isnan(got) & np.isnan(want))
        assert same.all(), (what, name, int((~same).sum()), np.argwhere(~same)[:3].tolist())


def _values(rng, shape, spread=True):
    x = rng.standard_normal(shape)
    if spread:
        x *= np.exp2(rng.integers(-6, 4, shape[:2]))[..., None]  # a size of its own for each token and head
    return x


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D,heads,bs,new,past", [
    (128, 2, 16, [1], [0]), (128, 3, 16, [1, 1, 1, 1, 1], [0, 1, 15, 16, 37]), (64, 2, 16, [33, 1, 0, 18], [7, 31, 5, 0]),
    (16, 5, 32, [5, 40, 70], [30, 0, 17]), (80, 1, 64, [100, 3], [3, 62]), (256, 2, 128, [130, 1, 1], [100, 127, 128]),
    (144, 1, 256, [300, 9], [250, 600]), (112, 9, 16, [3] * 20, list(range(20)))])
def test_write(device, fmt, dtype, D, heads, bs, new, past):
    """Twice: the second step appends to blocks that the first one left partly full, some with larger values (scales grow)."""
    rng = _rng("write", fmt, dtype, D, heads, bs)
    st = Step(rng, [2 * n for n in new], past, bs, padding=2)  # the tables for both steps
    st.new, st.starts = list(new), np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    c = kv8_ref.Cache(fmt, st.blocks, bs, heads, D, fill=rng)
    with Dev() as d:
        cache, at = _cache(d, c)
        for turn in range(2):
            st.T = int(st.starts[-1]) + 2
            k, k64 = _put(_values(rng, (st.T, heads, D)) * (1, 3)[turn], dtype)
            v, v64 = _put(_values(rng, (st.T, heads, D)) * (1, 0.5)[turn], dtype)
            log(f"kv8_write {dtype} {fmt} D={D} bs={bs} turn {turn}")
            native.kv8_write(dtype, d.put(k), d.put(v), cache, st.batch(d))
            native.synchronize()
            kv8_ref.write(c, k64, v64, st.starts, st.past, st.slots, st.pages)
            _check_write(d, c, at, turn)
            st.past = (st.past + np.int32(st.new)).astype(np.int32)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("layout", ["wide", "odd", "heads_first"])
def test_write_strides_and_alignment(device, fmt, dtype, layout):
    """K and V as views of a wider row, at odd addresses and strides, and as [heads, tokens, D]."""
    rng = _rng("strides", fmt, dtype, layout)
    D, heads, bs = 64, 3, 16
    st = Step(rng, [19, 2], [5, 40], bs)
    c = kv8_ref.Cache(fmt, st.blocks, bs, heads, D, fill=rng)
    size = np.dtype(NP[dtype]).itemsize
    if layout == "heads_first":
        raw, raw64 = _put(_values(rng, (2, heads, st.T * D), False), dtype)
        shape, st_t, st_h = (2, heads, st.T, D), D, st.T * D
        k64, v64 = raw64.reshape(shape).transpose(0, 2, 1, 3)
    else:
        row = 2 * heads * D + (16 if layout == "wide" else 3)
        raw, raw64 = _put(_values(rng, (1, st.T, row), False), dtype)
        st_t, st_h = row, D
        k64, v64 = (raw64[0, :, o:o + heads * D].reshape(st.T, heads, D) for o in (0, heads * D))
    with Dev() as d:
        cache, at = _cache(d, c)
        pad = size if layout == "odd" else 0
        p = d.put(raw, pad_bytes=pad)
        v = p + (heads * st.T * D if layout == "heads_first" else heads * D) * size
        log(f"kv8_write {layout} {dtype} {fmt}")
        native.kv8_write(dtype, p, v, cache, st.batch(d), k_stride_t=st_t, k_stride_h=st_h, v_stride_t=st_t, v_stride_h=st_h)
        native.synchronize()
        kv8_ref.write(c, k64, v64, st.starts, st.past, st.slots, st.pages)
        _check_write(d, c, at, layout)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_write_special_values(device, fmt, dtype):
    """Zeros, tiny and huge values, ties, NaN and infinities: each in a head of its own; then a block begun anew."""
    rng = _rng("special", fmt, dtype)
    D, bs = 32, 16
    heads = [0.0, 1e-30, 2.0 ** -50, 2.0 ** 46, 3e38, np.nan, np.inf, -np.inf, 1.0, 127.0, 448.0, -448.0 * 2.0 ** 40]
    st = Step(rng, [20, 20], [0, 7], bs)
    c = kv8_ref.Cache(fmt, st.blocks, bs, len(heads), D, fill=rng)
    x = rng.integers(-8, 9, (40, len(heads), D)) / 8.0
    for h, top in enumerate(heads):
        with np.errstate(invalid="ignore"):
            x[:, h] = x[:, h] * (top if np.isfinite(top) else 1.0)
        x[3::7, h, 5] = top
    with np.errstate(over="ignore"):
        k, k64 = _put(x, dtype)
        v, v64 = _put(x[::-1], dtype)
    with Dev() as d:
        cache, at = _cache(d, c)
        batch = st.batch(d)
        log(f"kv8_write special {dtype} {fmt}")
        native.kv8_write(dtype, d.put(k), d.put(v), cache, batch)
        native.synchronize()
        kv8_ref.write(c, k64, v64, st.starts, st.past, st.slots, st.pages)
        _check_write(d, c, at, "special")
        assert np.isnan(c.ks).any() and not np.isnan(c.ks[:, 8]).any()
        k, k64 = _put(rng.standard_normal(x.shape), dtype)  # finite values into the same places
        native.kv8_write(dtype, d.put(k), d.put(k), cache, batch)
        native.synchronize()
        kv8_ref.write(c, k64, k64, st.starts, st.past, st.slots, st.pages)
        _check_write(d, c, at, "again")


@pytest.mark.parametrize("bad", ["block", "negative", "slot", "past", "starts"])
def test_write_skips_what_does_not_fit(device, bad):
    rng = _rng("skip", bad)
    st = Step(rng, [5, 20, 3], [3, 10, 14], 16)
    if bad == "block":
        st.pages[st.slots[1], 1] = st.blocks
    elif bad == "negative":
        st.pages[st.slots[1], 0] = -7
    elif bad == "slot":
        st.slots[1] = len(st.pages)
    elif bad == "past":
        st.past[1] = st.pages.shape[1] * 16 - 19
    else:
        st.starts[3] = st.T + 1  # beyond the rows
    c = kv8_ref.Cache("i8", st.blocks, 16, 2, 32, fill=rng)
    k, k64 = _put(_values(rng, (st.T, 2, 32)), "f32")
    with Dev() as d:
        cache, at = _cache(d, c)
        log(f"kv8_write bad {bad}")
        native.kv8_write("f32", d.put(k), d.put(k), cache, st.batch(d))
        with pytest.raises(native.SlhipCacheError, match="outside the KV cache" if bad in ("block", "negative") else "does not fit"):
            native.synchronize()
        kv8_ref.write(c, k64, k64, st.starts, st.past, st.slots, st.pages)
        _check_write(d, c, at, bad)


# ---- attention -------------------------------------------------------------------------------------------------------

def _attend(d, dtype, st, c, q, G, *, max_new=0, work_pad=0, stream=None, y0=None, batch=None, cache=None, **kw):
    """Runs the attention on y filled with a pattern; returns y and the addresses."""
    H = c.heads * G
    cache = cache or _cache(d, c)[0]
    batch = batch or st.batch(d)
    need = native.kv8_attention_work_bytes(H, cache, batch, max_new)
    work = d.empty(max(need, 16), fill=0xFF)  # NaN bits: it needs no initialisation
    y = y0 if y0 is not None else d.empty(q.nbytes, fill=0x5A)
    native.kv8_attention(dtype, d.put(q), y, H, cache, batch, max_new=max_new, work=work, work_bytes=need, stream=stream, **kw)
    return y


def _check_y(got, want, bound, what, pattern=None):
    """Rows that are computed within the bound, the others left as they were."""
    done = ~np.isnan(bound).any(-1) | ~np.isnan(want).any(-1)
    with np.errstate(invalid="ignore"):
        off = np.abs(got - want)
    bad = done[..., None] & ~(off <= bound)
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:4].tolist(), float(np.nanmax(np.where(done[..., None], off / np.maximum(bound, 1e-300), 0))))
    if pattern is not None:
        assert (got[~done] == pattern).all() or (np.isnan(pattern) and np.isnan(got[~done]).all()), what


def _pattern(dtype):
    return _from(np.frombuffer(b"\x5a" * 4, NP[dtype])[:1], dtype)[0]


CASES = [  # D, heads, G, bs, new, past: one token to long, few rows and many, odd groups, requests without rows
    (128, 2, 4, 16, [1], [0]), (128, 2, 4, 16, [1], [63]), (128, 2, 4, 16, [1, 1, 1, 1], [64, 15, 0, 200]),
    (64, 1, 1, 32, [1, 1, 0, 1], [100, 31, 64, 1030]), (80, 2, 5, 16, [3, 1, 2], [37, 64, 0]), (16, 3, 8, 64, [2, 2], [63, 129]),
    (256, 1, 2, 128, [1, 6, 5], [300, 0, 127]), (112, 1, 16, 16, [1, 1], [5, 700]), (128, 1, 8, 16, [4, 3, 1], [90, 0, 500]),
    (128, 2, 4, 16, [70], [0]), (64, 2, 3, 16, [90, 40, 1, 0, 200], [0, 33, 500, 3, 64]), (144, 1, 1, 32, [65, 130], [100, 0]),
    (256, 1, 4, 256, [40, 1], [300, 10]), (96, 1, 40, 16, [1, 4], [77, 0]), (48, 1, 64, 16, [2, 3], [130, 5]), (128, 4, 1, 16, [129], [1]),
]


@pytest.mark.parametrize("fmt,dtype", [("i8", "f32"), ("e4m3", "f32"), ("i8", "bf16"), ("e4m3", "bf16")])
@pytest.mark.parametrize("D,heads,G,bs,new,past", CASES)
def test_attention(device, fmt, dtype, D, heads, G, bs, new, past):
    for max_new, wide in ((0, 500), (max(new), 1)):  # long table rows: contexts may be long, and heads are shared out
        rng = _rng("attn", fmt, dtype, D, heads, G, bs, tuple(new))
        st = Step(rng, new, past, bs, padding=3, wide=wide)
        c = kv8_ref.Cache(fmt, st.blocks, bs, heads, D, fill=rng)
        q, q64 = _put(rng.standard_normal((st.T, heads * G, D)) * 3, dtype)
        scale = 1 / np.sqrt(D)
        with Dev() as d:
            log(f"kv8_attention {dtype} {fmt} D={D} heads={heads}x{G} bs={bs} new={new} past={past} max_new={max_new} wide={wide}")
            y = _attend(d, dtype, st, c, q, G, max_new=max_new, scale=scale)
            native.synchronize()
            got = _from(d.get(y, q.shape, NP[dtype]), dtype)
        want, bound = kv8_ref.attention(c, q64, st.starts, st.past, st.slots, st.pages, scale=np.float32(scale).astype(float), dtype=dtype)
        _check_y(got, want, bound, f"max_new={max_new}", _pattern(dtype))


@pytest.mark.parametrize("fmt,dtype", [("i8", "f32"), ("e4m3", "bf16")])
@pytest.mark.parametrize("kw", [dict(softcap=20.0), dict(window=1), dict(window=17), dict(window=64), dict(window=100), dict(slopes=True),
                                dict(softcap=0.5, window=70, slopes=True), dict(scale=-0.3), dict(scale=0.0), dict(window=1 << 40)])
@pytest.mark.parametrize("D,heads,G,bs,new,past", [(64, 2, 4, 16, [1, 1, 3], [0, 300, 65]), (128, 1, 2, 32, [150, 20, 1], [0, 90, 333])])
def test_attention_scores(device, fmt, dtype, kw, D, heads, G, bs, new, past):
    """Caps, windows (of one key, inside a tile, at its border) and distance slopes."""
    rng = _rng("scores", fmt, dtype, str(kw), D)
    st = Step(rng, new, past, bs, wide=1 if dtype == "f32" else 200)
    c = kv8_ref.Cache(fmt, st.blocks, bs, heads, D, fill=rng)
    q, q64 = _put(rng.standard_normal((st.T, heads * G, D)) * 3, dtype)
    kw = {"scale": 0.125, **kw}
    slopes = np.exp2(-np.arange(1, heads * G + 1)).astype(np.float32) if kw.pop("slopes", False) else None
    with Dev() as d:
        log(f"kv8_attention scores {dtype} {fmt} {kw} slopes={slopes is not None} new={new}")
        y = _attend(d, dtype, st, c, q, G, slopes=None if slopes is None else d.put(slopes), **kw)
        native.synchronize()
        got = _from(d.get(y, q.shape, NP[dtype]), dtype)
    want, bound = kv8_ref.attention(c, q64, st.starts, st.past, st.slots, st.pages, dtype=dtype,
                                    slopes=None if slopes is None else slopes.astype(float), **{**kw, "scale": float(np.float32(kw["scale"]))})
    _check_y(got, want, bound, kw)


@pytest.mark.parametrize("fmt,dtype", [("e4m3", "f32"), ("i8", "bf16")])
@pytest.mark.parametrize("D,heads,G,bs,new,past", [
    (128, 2, 4, 16, [1], [9000]), (64, 1, 2, 64, [1, 1, 2], [20000, 3, 700]), (128, 1, 4, 32, [33, 100], [6000, 2000]), (256, 1, 1, 16, [20], [3000])])
def test_attention_long(device, fmt, dtype, D, heads, G, bs, new, past):
    """Contexts that are cut into ranges and joined, next to short ones that are not."""
    rng = _rng("long", fmt, dtype, D)
    st = Step(rng, new, past, bs)
    c = kv8_ref.Cache(fmt, st.blocks, bs, heads, D, fill=rng)
    q, q64 = _put(rng.standard_normal((st.T, heads * G, D)) * 2, dtype)
    with Dev() as d:
        log(f"kv8_attention long {dtype} {fmt} D={D} new={new} past={past}")
        y = _attend(d, dtype, st, c, q, G, scale=0.1, max_new=max(new))
        native.synchronize()
        got = _from(d.get(y, q.shape, NP[dtype]), dtype)
    want, bound = kv8_ref.attention(c, q64, st.starts, st.past, st.slots, st.pages, scale=float(np.float32(0.1)), dtype=dtype)
    _check_y(got, want, bound, "long")


@pytest.mark.parametrize("fmt,dtype", [("e4m3", "f32"), ("i8", "bf16")])
@pytest.mark.parametrize("window", [64, 1000, 1500, 2049, 3900])
@pytest.mark.parametrize("D,heads,G,new,past", [(64, 2, 4, [1, 2, 1], [4000, 1600, 5]), (128, 1, 2, [12, 16, 3], [3000, 0, 1501]),
                                                (256, 2, 2, [1, 8], [4100, 2000]), (64, 1, 2, [40, 1, 130], [4000, 3000, 1400])])
def test_attention_long_windows(device, fmt, dtype, window, D, heads, G, new, past):
    """Windows of many key tiles in longer contexts, whose borders lie inside tiles, ranges and blocks."""
    rng = _rng("windows", fmt, dtype, window, D)
    st = Step(rng, new, past, 32)
    c = kv8_ref.Cache(fmt, st.blocks, 32, heads, D, fill=rng)
    q, q64 = _put(rng.standard_normal((st.T, heads * G, D)) * 2, dtype)
    for max_new in (0, max(new)):
        with Dev() as d:
            log(f"kv8_attention long windows {dtype} {fmt} D={D} new={new} past={past} window={window} max_new={max_new}")
            y = _attend(d, dtype, st, c, q, G, scale=0.125, window=window, max_new=max_new)
            native.synchronize()
            got = _from(d.get(y, q.shape, NP[dtype]), dtype)
        want, bound = kv8_ref.attention(c, q64, st.starts, st.past, st.slots, st.pages, scale=0.125, window=window, dtype=dtype)
        _check_y(got, want, bound, f"max_new={max_new}")


@pytest.mark.parametrize("fmt,dtype", [("i8", "bf16"), ("e4m3", "f32")])
@pytest.mark.parametrize("B,heads,longest,wide", [(40, 16, 1900, 1), (70, 16, 3000, 1), (20, 4, 900, 1), (20, 4, 900, 200)])
@pytest.mark.parametrize("D,G,new", [(64, 4, 1), (128, 2, 12), (256, 3, 2)])
def test_attention_of_uneven_contexts(device, fmt, dtype, B, heads, longest, wide, D, G, new):
    """Steps of many heads with a thread block each, and with a shared line; one context is as long as may be."""
    rng = _rng("uneven", fmt, dtype, B, D)
    past = np.where(rng.random(B) < 0.1, longest, rng.integers(0, 100, B))
    past[3] = longest
    st = Step(rng, [new] * B, past, 16, wide=wide)
    c = kv8_ref.Cache(fmt, st.blocks, 16, heads, D, fill=rng)
    q, q64 = _put(rng.standard_normal((st.T, heads * G, D)) * 2, dtype)
    with Dev() as d:
        log(f"kv8_attention uneven {dtype} {fmt} B={B} heads={heads} D={D} G={G} new={new} longest={longest} wide={wide}")
        y = _attend(d, dtype, st, c, q, G, scale=0.125, max_new=new)
        native.synchronize()
        got = _from(d.get(y, q.shape, NP[dtype]), dtype)
    want, bound = kv8_ref.attention(c, q64, st.starts, st.past, st.slots, st.pages, scale=0.125, dtype=dtype)
    _check_y(got, want, bound, "uneven")


@pytest.mark.parametrize("fmt,dtype,G,most", [("i8", "f32", 2, 1), ("e4m3", "bf16", 4, 7), ("e4m3", "bf16", 1, 40)])
@pytest.mark.parametrize("B,wide", [(64, 80), (65, 1), (70, 80), (300, 80), (4500, 1)])
def test_many_requests(device, fmt, dtype, G, most, B, wide):
    """More requests than lanes of a wave, and than its square: the write and the attention find theirs. Some bring nothing."""
    rng = _rng("many", fmt, dtype, B)
    new = rng.integers(0, 3, B)
    new[rng.integers(0, B, 20)] = most
    new = np.minimum(new, most)
    st = Step(rng, new.tolist(), rng.integers(0, 60, B) * (rng.random(B) < 0.8), 16, padding=2, wide=wide)
    c = kv8_ref.Cache(fmt, st.blocks, 16, 2, 32, fill=rng)
    q, q64 = _put(rng.standard_normal((st.T, 2 * G, 32)) * 3, dtype)
    k, k64 = _put(_values(rng, (st.T, 2, 32)), dtype)
    v, v64 = _put(_values(rng, (st.T, 2, 32)), dtype)
    with Dev() as d:
        cache, at = _cache(d, c)
        batch = st.batch(d)
        log(f"{B} requests, {dtype} {fmt} G={G} most={most} wide={wide}")
        native.kv8_write(dtype, d.put(k), d.put(v), cache, batch)
        native.synchronize()
        kv8_ref.write(c, k64, v64, st.starts, st.past, st.slots, st.pages)
        _check_write(d, c, at, B)
        for max_new in (0, most):
            y = _attend(d, dtype, st, c, q, G, batch=batch, cache=cache, scale=0.125, max_new=max_new)
            native.synchronize()
            got = _from(d.get(y, q.shape, NP[dtype]), dtype)
            want, bound = kv8_ref.attention(c, q64, st.starts, st.past, st.slots, st.pages, scale=0.125, dtype=dtype)
            _check_y(got, want, bound, f"max_new={max_new}", _pattern(dtype))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("new,past", [([1, 2, 1], [40, 100, 3]), ([60, 70], [40, 10])])
def test_attention_scales_far_apart(device, dtype, new, past):
    """Blocks whose V scales lie 2^60 apart: weights count with their scale, and a zero-valued block keeps its weight."""
    rng = _rng("far", dtype, len(new))
    st = Step(rng, new, past, 16)
    c = kv8_ref.Cache("e4m3", st.blocks, 16, 2, 64, fill=rng)
    c.vs[:] = np.exp2(rng.integers(-40, 21, c.vs.shape)).astype(np.float32)
    c.vs[::3], c.v[::3] = 2.0 ** -40, 0
    c.ks[:] = np.exp2(rng.integers(-12, -6, c.ks.shape)).astype(np.float32)
    q, q64 = _put(rng.standard_normal((st.T, 4, 64)) * np.exp2(rng.integers(-60, 4, (st.T, 4, 1))), dtype)
    q[0, 0], q64[0, 0] = 0, 0
    with Dev() as d:
        log(f"kv8_attention scales far apart {dtype}")
        y = _attend(d, dtype, st, c, q, 2, scale=0.2)
        native.synchronize()
        got = _from(d.get(y, q.shape, NP[dtype]), dtype)
    want, bound = kv8_ref.attention(c, q64, st.starts, st.past, st.slots, st.pages, scale=float(np.float32(0.2)), dtype=dtype)
    _check_y(got, want, bound, "far apart")


def test_as_many_requests_as_there_may_be(device):
    """65536 requests, of which a few hundred bring rows, the first and the last among them."""
    rng = _rng("most")
    B = 65536
    new, past = np.zeros(B, int), np.zeros(B, int)
    at = np.concatenate([[0, 63, 64, 4095, 4096, B - 1], rng.integers(0, B, 300)])
    new[at], past[at] = rng.integers(1, 4, len(at)), rng.integers(0, 100, len(at))
    st = Step(rng, new.tolist(), past, 16, padding=1, wide=80)
    c = kv8_ref.Cache("i8", st.blocks, 16, 1, 32, fill=rng)
    q, q64 = _put(rng.standard_normal((st.T, 4, 32)) * 2, "bf16")
    k, k64 = _put(_values(rng, (st.T, 1, 32)), "bf16")
    with Dev() as d:
        cache, where = _cache(d, c)
        batch = st.batch(d)
        log(f"{B} requests, {st.T} rows")
        native.kv8_write("bf16", d.put(k), d.put(k), cache, batch)
        native.synchronize()
        kv8_ref.write(c, k64, k64, st.starts, st.past, st.slots, st.pages)
        _check_write(d, c, where, B)
        y = _attend(d, "bf16", st, c, q, 4, batch=batch, cache=cache, scale=0.125, max_new=3)
        native.synchronize()
        got = _from(d.get(y, q.shape, np.uint16), "bf16")
    want, bound = kv8_ref.attention(c, q64, st.starts, st.past, st.slots, st.pages, scale=0.125, dtype="bf16")
    _check_y(got, want, bound, B, _pattern("bf16"))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("slopes", [False, True])
@pytest.mark.parametrize("new,past", [([1, 2], [130, 500]), ([40, 50], [130, 500])])
def test_attention_of_large_scores(device, dtype, slopes, new, past):
    """Scores of up to 2^60: far past where f32 tells neighbours apart, but the largest of a row is larger by a third, so its
    key's value is the answer. (Weights of e^-1000 and less for the others: the rest is y's rounding, and 2^-11 or 2^-22 of it for
    the weight, which cancels.)"""
    rng = _rng("large", dtype, slopes, len(new))
    st = Step(rng, new, past, 16)
    D, heads, G = 64, 2, 2
    c = kv8_ref.Cache("i8", st.blocks, 16, heads, D, fill=rng)
    c.k[:], c.ks[:], c.vs[:] = 0, 1.0, 1.0
    c.k[..., 0] = 90
    best = [int(rng.integers(0, p + 1)) for p in past]  # every row of the request sees it
    for i, s in enumerate(st.slots):
        c.k[st.pages[s, best[i] // 16], :, best[i] % 16, 0] = 120
    q = np.zeros((st.T, heads * G, D))
    q[..., 0] = np.exp2(rng.integers(5, 54, (st.T, heads * G)))
    bits, _ = _put(q, dtype)
    with Dev() as d:
        log(f"kv8_attention large scores {dtype} slopes={slopes} new={new}")
        y = _attend(d, dtype, st, c, bits, G, scale=1.0, slopes=d.put(np.full(heads * G, 0.25, np.float32)) if slopes else None)
        native.synchronize()
        got = _from(d.get(y, bits.shape, NP[dtype]), dtype)
    for i, s in enumerate(st.slots):
        v = c.v.view(np.int8)[st.pages[s, best[i] // 16], :, 0, :, best[i] % 16].astype(np.float64)  # [heads, D]
        rows = got[st.starts[i]:st.starts[i + 1]].reshape(-1, heads, G, D)
        assert (np.abs(rows - v[None, :, None]) <= np.abs(v[None, :, None]) * 2.0 ** (-20 if dtype == "f32" else -7)).all(), i


@pytest.mark.parametrize("fmt,dtype", [("e4m3", "f32"), ("e4m3", "bf16"), ("i8", "bf16")])
@pytest.mark.parametrize("new,past", [([1, 1], [70, 10]), ([40, 50], [70, 0])])
def test_attention_does_not_see_what_is_not_there(device, fmt, dtype, new, past):
    """Codes behind a request's last token, blocks of nobody and their scales may hold anything; a poisoned block gives NaN
    to the rows that see it and to no others."""
    rng = _rng("unseen", fmt, dtype, len(new))
    st = Step(rng, new, past, 16, wide=1 if dtype == "f32" else 300)
    c = kv8_ref.Cache(fmt, st.blocks, 16, 2, 64, fill=rng)
    want, bound = None, None
    q, q64 = _put(rng.standard_normal((st.T, 4, 64)), dtype)
    want, bound = kv8_ref.attention(c, q64, st.starts, st.past, st.slots, st.pages, scale=0.25, dtype=dtype)
    used = set()
    for i, s in enumerate(st.slots):
        n = int(st.past[i]) + st.new[i]
        ids = st.pages[s, :-(-n // 16)]
        used |= set(ids.tolist())
        if n % 16:
            c.k[ids[-1], :, n % 16:] = 0x7F
            c.v[ids[-1], :, :, :, n % 16:] = 0xFF
    for b in set(range(st.blocks)) - used:
        c.k[b], c.v[b], c.ks[b], c.vs[b] = 0x7F, 0x7F, np.nan, np.inf
    with Dev() as d:
        log(f"kv8_attention unseen {dtype} {fmt} new={new}")
        y = _attend(d, dtype, st, c, q, 2, scale=0.25)
        native.synchronize()
        _check_y(_from(d.get(y, q.shape, NP[dtype]), dtype), want, bound, "unseen")
        # request 0's block of tokens 32..47 loses its scale, in head 1
        block = st.pages[st.slots[0], 2]
        for name in ("ks", "vs"):
            p = c.copy()
            getattr(p, name)[block, 1] = np.nan
            y = _attend(d, dtype, st, p, q, 2, scale=0.25)
            native.synchronize()
            got = _from(d.get(y, q.shape, NP[dtype]), dtype)
            lost = np.zeros((st.T, 4), bool)
            lost[:st.new[0], 2:] = True  # all of request 0's rows come after token 47
            assert np.isnan(got[lost]).all(), name
            _check_y(np.where(lost[..., None], want, got), want, bound, name)
            y = _attend(d, dtype, st, p, q, 2, scale=0.25, window=20)  # rows from position 67 on do not see token 47
            native.synchronize()
            got = _from(d.get(y, q.shape, NP[dtype]), dtype)
            w2, b2 = kv8_ref.attention(c, q64, st.starts, st.past, st.slots, st.pages, scale=0.25, dtype=dtype, window=20)
            _check_y(got, w2, b2, name + " out of the window")


@pytest.mark.parametrize("new", [[1, 2, 1], [30, 40, 20]])
@pytest.mark.parametrize("bad", ["block", "all_blocks", "slot", "past", "max_new"])
def test_attention_of_what_does_not_fit(device, new, bad):
    """Keys of blocks outside the cache are not seen (a row without keys is 0); rows of requests that do not fit stay."""
    rng = _rng("unfit", bad, len(new))
    st = Step(rng, new, [40, 50, 20], 16, wide=1 if bad == "slot" else 300)
    max_new = 0
    if bad == "block":
        st.pages[st.slots[1], 1] = -1
        st.pages[st.slots[2], 0] = st.blocks
    elif bad == "all_blocks":
        st.pages[st.slots[1]] = 1 << 30
    elif bad == "slot":
        st.slots[1] = -1
    elif bad == "past":
        st.past[1] = -5
    else:
        max_new = max(new) - 1
    c = kv8_ref.Cache("i8", st.blocks, 16, 1, 32, fill=rng)
    q, q64 = _put(rng.standard_normal((st.T, 2, 32)), "f32")
    want, bound = kv8_ref.attention(c, q64, st.starts, st.past, st.slots, st.pages, scale=0.3)
    if bad == "max_new":
        i = new.index(max(new))
        want[st.starts[i]:st.starts[i + 1]] = bound[st.starts[i]:st.starts[i + 1]] = np.nan
    with Dev() as d:
        log(f"kv8_attention unfit {bad} new={new}")
        y = _attend(d, "f32", st, c, q, 2, scale=0.3, max_new=max_new)
        with pytest.raises(native.SlhipCacheError, match="outside the KV cache" if "block" in bad else "does not fit"):
            native.synchronize()
        got = d.get(y, q.shape, np.float32).astype(np.float64)
    _check_y(got, want, bound, bad, _pattern("f32"))
    if bad == "all_blocks":
        assert (got[st.starts[1]:st.starts[2]] == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("layout", ["wide", "odd", "heads_first", "in_place"])
@pytest.mark.parametrize("new,past", [([1, 3], [30, 70]), ([50, 9], [30, 70])])
def test_attention_strides(device, dtype, layout, new, past):
    rng = _rng("attn strides", dtype, layout, len(new))
    D, heads, G = 48, 2, 3
    H = heads * G
    st = Step(rng, new, past, 16)
    c = kv8_ref.Cache("e4m3", st.blocks, 16, heads, D, fill=rng)
    size, T = np.dtype(NP[dtype]).itemsize, st.T
    shape, kw, pad = (T, H, D), {}, 0
    if layout == "heads_first":
        shape, kw = (H, T, D), dict(q_stride_t=D, q_stride_h=T * D, y_stride_t=D, y_stride_h=T * D)
    elif layout != "in_place":
        row = H * D + (32 if layout == "wide" else 5)
        shape, kw, pad = (T, row), dict(q_stride_t=row, y_stride_t=row), size if layout == "odd" else 0
    raw, raw64 = _put(rng.standard_normal(shape), dtype)
    as_rows = lambda x: x.transpose(1, 0, 2) if layout == "heads_first" else x[:, :H * D].reshape(T, H, D) if len(shape) == 2 else x  # noqa: E731
    want, bound = kv8_ref.attention(c, as_rows(raw64), st.starts, st.past, st.slots, st.pages, scale=0.25, dtype=dtype)
    with Dev() as d:
        cache, batch = _cache(d, c)[0], st.batch(d)
        need = native.kv8_attention_work_bytes(H, cache, batch, 0)
        q = d.put(raw, pad_bytes=pad)
        y = q if layout == "in_place" else d.empty(raw.nbytes, pad_bytes=pad, fill=0x5A)
        log(f"kv8_attention {layout} {dtype} new={new}")
        native.kv8_attention(dtype, q, y, H, cache, batch, scale=0.25, work=d.empty(need), work_bytes=need, **kw)
        native.synchronize()
        got = _from(d.get(y, shape, NP[dtype]), dtype)
    _check_y(as_rows(got), want, bound, layout)
    if len(shape) == 2:
        assert (got[:, H * D:] == _pattern(dtype)).all()


def test_offsets_past_32_bits(device):
    """A cache of 2.3 GB a side whose requests lie at its end: block, code and scale offsets pass 2^31."""
    rng = _rng("offsets")
    D, heads, bs = 256, 4, 16
    blocks = (1 << 31) // (heads * bs * D) + 9000
    st = Step(rng, [1, 40], [30, 20], bs)
    small = kv8_ref.Cache("i8", st.blocks, bs, heads, D, fill=rng)
    base = blocks - st.blocks
    pages = np.where(st.pages >= 0, st.pages + base, -1).astype(np.int32)
    q, q64 = _put(rng.standard_normal((st.T, 8, D)), "bf16")
    k, k64 = _put(_values(rng, (st.T, heads, D)), "bf16")
    with Dev() as d:
        n = blocks * heads * bs * D
        log(f"cache of 2 x {n} bytes")
        ck, cv = d.empty(n, fill=None), d.empty(n, fill=None)
        cks, cvs = d.empty(blocks * heads * 4, fill=None), d.empty(blocks * heads * 4, fill=None)
        o, so = base * heads * bs * D, base * heads * 4
        for at, x in ((ck + o, small.k), (cv + o, small.v), (cks + so, small.ks), (cvs + so, small.vs)):
            native.call("slhip_memcpy_h2d", at, np.ascontiguousarray(x).ctypes.data, x.nbytes, None)
            native.synchronize()
        cache = native.kv8_cache("i8", ck, cv, cks, cvs, blocks, bs, heads, D)
        st.pages = pages
        batch = st.batch(d)
        native.kv8_write("bf16", d.put(k), d.put(k), cache, batch)
        native.synchronize()
        st.pages = np.where(pages >= 0, pages - base, -1).astype(np.int32)
        kv8_ref.write(small, k64, k64, st.starts, st.past, st.slots, st.pages)
        _check_write(d, small, (ck + o, cv + o, cks + so, cvs + so), "far blocks")
        y = _attend(d, "bf16", st, small, q, 2, batch=batch, cache=cache, scale=0.1)
        native.synchronize()
        got = _from(d.get(y, q.shape, np.uint16), "bf16")
    want, bound = kv8_ref.attention(small, q64, st.starts, st.past, st.slots, st.pages, scale=float(np.float32(0.1)), dtype="bf16")
    _check_y(got, want, bound, "far blocks")


# ---- together ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("fmt,dtype", [("e4m3", "bf16"), ("i8", "f32")])
def test_serving_steps(device, captured, fmt, dtype):
    """A prompt step and decode steps as a program runs them: tables, rope of K, write, attention; the decode steps eager, or
    one captured graph replayed with new lengths and inputs. Then requests end and their blocks come back."""
    rng = _rng("steps", fmt, dtype)
    B, heads, G, D, bs, bps = 5, 2, 2, 64, 16, 12
    H, blocks = heads * G, 40
    prompt = [33, 1, 70, 16, 47]
    tmax = sum(prompt) + 5
    c = kv8_ref.Cache(fmt, blocks, bs, heads, D)
    pages, free, n_free = np.full((8, bps), -1, np.int32), rng.permutation(blocks).astype(np.int32), blocks
    slots = rng.permutation(8)[:B].astype(np.int32)
    past = np.zeros(B, np.int32)
    size = np.dtype(NP[dtype]).itemsize
    st = native.Stream()
    with Dev() as d:
        cache, at = _cache(d, c)
        dev = {"past": d.put(past), "count": d.put(np.int32(prompt)), "slots": d.put(slots), "pages": d.put(pages), "free": d.put(free),
               "n": d.put(np.int32([n_free])), "starts": d.empty(4 * (B + 1)), "seq": d.empty(16 * tmax), "pos": d.empty(4 * tmax),
               "q": d.empty(tmax * H * D * size), "k": d.empty(tmax * heads * D * size), "kr": d.empty(tmax * heads * D * size, fill=0),
               "v": d.empty(tmax * heads * D * size), "y": d.empty(tmax * H * D * size)}

        def step(tokens, max_new):
            kp = native.kv_pages(B, dev["past"], dev["count"], dev["pages"], 8, bps, bs, dev["free"], blocks, dev["n"], dev["n"], tokens,
                                 dev["starts"], seq=dev["seq"], pos=dev["pos"], slots=dev["slots"])
            batch = native.kv8_batch(B, tokens, dev["starts"], dev["past"], dev["pages"], 8, bps, slots=dev["slots"])
            need = native.kv8_attention_work_bytes(H, cache, batch, max_new)
            work = d.empty(need)

            def run():
                s = st.handle
                native.kv_pages_advance(kp, stream=s)
                native.rope(dtype, dtype, [dict(x=dev["k"], y=dev["kr"], heads=heads)], dev["pos"], tokens, D, base=1e4, stream=s)
                native.kv8_write(dtype, dev["kr"], dev["v"], cache, batch, stream=s)
                native.kv8_attention(dtype, dev["q"], dev["y"], H, cache, batch, scale=0.125, max_new=max_new, work=work, work_bytes=need, stream=s)
            return run

        def upload(name, x):
            native.call("slhip_memcpy_h2d", dev[name], np.ascontiguousarray(x).ctypes.data, x.nbytes, st.handle)
            st.sync()

        decode, graph = step(B, 1), None
        for turn in range(6):
            count = prompt if turn == 0 else [1] * B
            if turn == 4:
                count = [1, 0, 1, 1, 0]  # two requests pause: rows behind the last are padding
            tokens = tmax if turn == 0 else B
            host = {}
            for name, n in (("q", H), ("k", heads), ("v", heads)):
                bits, host[name] = _put(rng.standard_normal((tokens, n, D)) * (1 + turn), dtype)
                upload(name, bits)
            upload("past", past)
            upload("count", np.int32(count))
            native.call("slhip_memset", dev["y"], 0x5A, tmax * H * D * size, st.handle)
            st.sync()
            log(f"serving step {turn} captured={captured} {fmt} {dtype}")
            if turn == 0:
                step(tmax, max(prompt))()
            elif captured:
                graph = graph or native.Graph(st, decode)
                graph.launch(st)
            else:
                decode()
            st.sync()
            want = kv8_ref.advance(past, count, slots, pages, bs, free, n_free, tokens)
            assert want[0]
            ok, pages, n_free, starts, seq, pos = want
            assert np.array_equal(d.get(dev["pages"], pages.shape, np.int32), pages)
            assert np.array_equal(d.get(dev["seq"], (tokens, 4), np.int32), seq)
            assert d.get(dev["n"], (1,), np.int32)[0] == n_free
            kr = _from(d.get(dev["kr"], (tokens, heads, D), NP[dtype]), dtype)  # rope has tests of its own
            kv8_ref.write(c, kr, host["v"], starts, past, slots, pages)
            _check_write(d, c, at, turn)
            got = _from(d.get(dev["y"], (tokens, H, D), NP[dtype]), dtype)
            y, bound = kv8_ref.attention(c, host["q"], starts, past, slots, pages, scale=0.125, dtype=dtype)
            _check_y(got, y, bound, f"turn {turn}", _pattern(dtype))
            past = (past + np.int32(count)).astype(np.int32)
        rel = native.kv_pages(2, d.put(past[1:3]), None, dev["pages"], 8, bps, bs, dev["free"], blocks, dev["n"], dev["n"], slots=d.put(slots[1:3]))
        log("kv_pages_release of two requests")
        native.kv_pages_release(rel, stream=st.handle)
        st.sync()
        ok, pages, free, n_free = kv8_ref.release(past[1:3], slots[1:3], pages, bs, free, n_free)
        assert ok and np.array_equal(d.get(dev["pages"], pages.shape, np.int32), pages)
        assert np.array_equal(d.get(dev["free"], free.shape, np.int32), free) and d.get(dev["n"], (1,), np.int32)[0] == n_free
        graph = None


@pytest.mark.parametrize("dtype,D,max_new", [("bf16", 256, 0), ("f32", 128, 0), ("bf16", 128, 8)])
def test_captured_attention_with_other_lengths(device, dtype, D, max_new):
    """One captured call of room for many rows and long contexts, replayed with other lengths, among them none at all, and the
    program's own work in between: what an eager call gives, and the statement's values."""
    rng = _rng("captured", dtype, D, max_new)
    B, heads, G, bs, rows = 3, 2, 4, 16, 120
    top = Step(rng, [rows, rows, rows], [2000, 2000, 2000], bs)
    c = kv8_ref.Cache("i8", top.blocks, bs, heads, D, fill=rng)
    lengths = [([1, 1, 1], [1700, 3, 900]), ([8, 5, 1], [0, 1999, 64]), ([0, 0, 0], [5, 6, 7]), ([1, 8, 0], [31, 32, 33])]
    if not max_new:
        lengths += [([100, 3, 17], [0, 2000, 300]), ([1, 40, 60], [2000, 10, 0])]
    st = native.Stream()
    with Dev() as d:
        cache, batch = _cache(d, c)[0], top.batch(d)
        starts, past = top.dev[:2]
        batch = native.kv8_batch(B, rows, starts, past, top.dev[2], top.pages.shape[0], top.pages.shape[1], slots=top.dev[3])
        q, q64 = _put(rng.standard_normal((rows, heads * G, D)) * 2, dtype)
        pq, y, eager = d.put(q), d.empty(q.nbytes), d.empty(q.nbytes)
        need = native.kv8_attention_work_bytes(heads * G, cache, batch, max_new)
        work = d.empty(max(need, 16), fill=0xFF)

        def run(out=y, stream=st.handle):
            native.kv8_attention(dtype, pq, out, heads * G, cache, batch, scale=0.0625, max_new=max_new, work=work, work_bytes=need, stream=stream)

        graph = native.Graph(st, run)
        for turn, (new, old) in enumerate(lengths * 2):
            s = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
            for at, x in ((starts, s), (past, np.int32(old))):
                native.call("slhip_memcpy_h2d", at, np.ascontiguousarray(x).ctypes.data, x.nbytes, st.handle)
            for out in (y, eager):
                native.call("slhip_memset", out, 0x5A, q.nbytes, st.handle)
            st.sync()
            log(f"captured attention {dtype} D={D} turn {turn}: new={new} past={old}")
            graph.launch(st)
            st.sync()
            run(eager)
            st.sync()
            got = d.get(y, q.shape, NP[dtype])
            assert np.array_equal(got, d.get(eager, q.shape, NP[dtype])), turn
            if turn < len(lengths):
                want, bound = kv8_ref.attention(c, q64, s, np.int32(old), top.slots, top.pages, scale=0.0625, dtype=dtype)
                _check_y(_from(got, dtype), want, bound, turn, _pattern(dtype))
        graph = None


def test_two_streams_at_once(device):
    """Overlapping calls with workspaces of their own, on two streams, several times: the same bits as one after another."""
    rng = _rng("streams")
    st = Step(rng, [1, 1, 40], [3000, 500, 100], 16)
    c = kv8_ref.Cache("e4m3", st.blocks, 16, 2, 128, fill=rng)
    q, _ = _put(rng.standard_normal((st.T, 8, 128)), "bf16")
    with Dev() as d:
        cache, batch = _cache(d, c)[0], st.batch(d)
        need = native.kv8_attention_work_bytes(8, cache, batch, 0)
        pq, streams = d.put(q), [native.Stream(), native.Stream()]
        ys, works = [d.empty(q.nbytes) for _ in range(3)], [d.empty(need) for _ in range(2)]
        native.kv8_attention("bf16", pq, ys[2], 8, cache, batch, scale=0.1, work=works[0], work_bytes=need)
        native.synchronize()
        for rep in range(3):
            log(f"two streams, turn {rep}")
            for i in range(2):
                native.kv8_attention("bf16", pq, ys[i], 8, cache, batch, scale=0.1, work=works[i], work_bytes=need, stream=streams[i].handle)
            for s in streams:
                s.sync()
            one = d.get(ys[2], q.shape, np.uint16)
            for i in range(2):
                assert np.array_equal(d.get(ys[i], q.shape, np.uint16), one)
