"""GPU parity of the adapters of many requests (slhip_lora) against the 64-bit statement of tests/step_ref.py, within the bound
derived there; rows that no request has stay bit for bit as they were."""
import zlib

import numpy as np
import pytest

import oracle
from sharplight_amd import native
from tests import step_ref
from tests.devutil import Dev, log

pytestmark = pytest.mark.gpu

NP = {"f32": np.float32, "bf16": np.uint16, "f16": np.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def rng_of(*parts):
    return np.random.default_rng(zlib.crc32(repr(parts).encode()))


def held(x, dtype):
    """f64 values as an array of the dtype, and the values it then holds."""
    with np.errstate(over="ignore"):
        f = x.astype(np.float32)
        if dtype == "f32":
            return f, f.astype(np.float64)
        if dtype == "f16":
            return f.astype(np.float16), f.astype(np.float16).astype(np.float64)
    b = oracle.to_bf16(f)
    return b, oracle.from_bf16(b).astype(np.float64)


def values(bits, dtype):
    return (oracle.from_bf16(bits) if dtype == "bf16" else bits).astype(np.float64)


def wide(x, stride, fill):
    """Rows of a larger array, its other places `fill`."""
    out = np.full((len(x), stride), fill, x.dtype)
    out[:, :x.shape[1]] = x
    return out


class Case:
    """Inputs on the host, and what slhip_lora makes of them."""

    def __init__(self, name, new, adapter, adapters, rank, K, N, x="f32", w="f32", y="f32", ranks=None, scale=None, add=True, padding=0):
        rng = rng_of(name, len(new), K, N, rank, x, w, y)
        self.new, self.starts = list(new), np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.adapter, self.adapters, self.rank, self.K, self.N = np.int32(adapter), adapters, rank, K, N
        self.T = int(self.starts[-1]) + padding
        self.dx, self.dw, self.dy = x, w, y
        self.x, self.vx = held(rng.standard_normal((self.T, K)), x)
        self.a, self.va = held(rng.standard_normal((adapters, rank, K)) / np.sqrt(K), w)
        self.b, self.vb = held(rng.standard_normal((adapters, N, rank)) / np.sqrt(rank), w)
        self.add, self.vadd = held(rng.standard_normal((self.T, N)), y) if add else (None, None)
        self.ranks, self.scale = ranks, scale

    def expected(self):
        return step_ref.lora(self.vx, self.vadd, self.va, self.vb, self.starts, self.adapter, self.ranks, self.scale,
                             bf16_parts=self.dy == "bf16")

    def put(self, d, in_place=False, shift=0, x_stride=None, add_stride=None, y_stride=None, a_pad=0, b_pad=0):
        """The call's arguments; strides, shifts (elements) and gaps as asked, every gap a NaN."""
        nan = {"f32": np.float32(np.nan), "f16": np.float16(np.nan), "bf16": np.uint16(0x7FC1)}
        flat = lambda v, pad: wide(v.reshape(len(v), -1), v[0].size + pad, nan[self.dw])  # noqa: E731
        xs, ys = x_stride or self.K, y_stride or self.N
        as_ = ys if in_place else add_stride or self.N
        px = d.put(wide(self.x, xs, nan[self.dx]), pad_bytes=shift * SIZE[self.dx])
        pa, pb = (d.put(flat(v, pad), pad_bytes=shift * SIZE[self.dw]) for v, pad in ((self.a, a_pad), (self.b, b_pad)))
        self.before = np.full((self.T, ys), 0xAB * 0x0101, np.uint16).astype(NP["bf16"]) if self.dy == "bf16" else np.full((self.T, ys), -777.25, np.float32)
        if in_place:
            self.before[:, :self.N] = self.add
        py = d.put(self.before, pad_bytes=shift * SIZE[self.dy])
        padd = py if in_place else None if self.add is None else d.put(wide(self.add, as_, nan[self.dy]), pad_bytes=shift * SIZE[self.dy])
        self.py, self.ys = py, ys
        sets = native.lora_set(self.dw, pa, pb, self.adapters, self.rank, self.K, self.N, rank=None if self.ranks is None else d.put(np.int32(self.ranks)),
                               scale=None if self.scale is None else d.put(np.float32(self.scale)),
                               a_stride=self.rank * self.K + a_pad, b_stride=self.rank * self.N + b_pad)
        rows = native.lora_rows(len(self.new), self.T, d.put(self.starts), d.put(self.adapter))
        size = native.lora_work_bytes(self.T, self.rank)
        return (self.dx, self.dy, px, padd, py, sets, rows), dict(x_stride=xs, add_stride=as_, y_stride=ys, work=d.empty(max(size, 16)), work_bytes=size)

    def check(self, d, got=None):
        got = d.get(self.py, (self.T, self.ys), NP[self.dy]) if got is None else got
        y, bound = self.expected()
        bound = step_ref.rounded_bound(y, bound, self.dy)
        inside = ~np.isnan(y)
        whole = np.zeros(got.shape, bool)
        whole[:, :self.N] = inside
        kept = got.view(np.uint32 if self.dy == "f32" else np.uint16)[~whole], self.before.view(np.uint32 if self.dy == "f32" else np.uint16)[~whole]
        assert np.array_equal(*kept), "places outside the rows and outputs were written"
        v = values(got[:, :self.N], self.dy)
        off = np.abs(v - y)[inside]
        worst = np.max(off / np.maximum(bound[inside], 1e-300)) if off.size else 0.0
        assert np.all(off <= bound[inside]), worst
        return v


def run(d, case, **kw):
    args, more = case.put(d, **kw)
    log(f"lora new={case.new[:6]}.. T={case.T} adapters={case.adapters} rank={case.rank} K={case.K} N={case.N} {case.dx}/{case.dw}/{case.dy} {kw}")
    native.lora(*args, **more)
    native.synchronize()
    return case.check(d)


TYPES = [("bf16", "bf16", "bf16"), ("f32", "bf16", "f32"), ("f32", "f32", "f32"), ("f32", "f16", "f32"), ("bf16", "f16", "bf16"),
         ("bf16", "bf16", "f32"), ("f32", "bf16", "bf16"), ("bf16", "f32", "bf16")]


@pytest.mark.parametrize("x,w,y", TYPES)
@pytest.mark.parametrize("new,rank,K,N", [
    ([1], 16, 512, 256), ([1], 1, 8, 8), ([2], 3, 9, 11), ([5], 8, 64, 64), ([17], 16, 100, 70), ([70], 24, 257, 131), ([200], 64, 320, 300), ([40], 100, 130, 65),
    ([64], 256, 192, 257)])
def test_one_request(device, new, rank, K, N, x, w, y):
    with Dev() as d:
        run(d, Case("one", new, [1], 3, rank, K, N, x, w, y))


@pytest.mark.parametrize("x,w,y", TYPES[:4])
@pytest.mark.parametrize("B,most,adapters,rank,K,N", [
    (2, 1, 1, 8, 128, 96), (16, 1, 16, 16, 256, 512), (64, 1, 5, 16, 640, 200), (65, 3, 4, 32, 96, 72), (300, 1, 7, 16, 128, 130),
    (23, 40, 6, 24, 200, 264), (7, 150, 3, 16, 384, 320), (600, 5, 3, 8, 64, 64), (9, 300, 2, 48, 72, 136)])
def test_many_requests(device, B, most, adapters, rank, K, N, x, w, y):
    rng = rng_of("many", B, most)
    new = rng.integers(0 if most > 1 else 1, most + 1, B)
    if new.sum() == 0:
        new[0] = 1
    adapter = rng.integers(-1, adapters, B)
    ranks = rng.integers(0, rank + 1, adapters)
    ranks[0] = rank
    with Dev() as d:
        run(d, Case("many", new, adapter, adapters, rank, K, N, x, w, y, ranks=ranks, scale=rng.standard_normal(adapters), padding=int(rng.integers(0, 20))))


@pytest.mark.parametrize("B,most,adapters,share", [(65, 1, 70, 0.0), (66, 700, 3, 0.8), (130, 40, 1, 0.3), (1000, 3, 400, 0.0), (2500, 2, 900, 0.5)])
def test_lists_of_tiles(device, B, most, adapters, share):
    """More than 64 requests: few and many adapters, long and empty requests."""
    rng = rng_of("lists", B, most, adapters)
    new = np.where(rng.random(B) < share, 0, rng.integers(1, most + 1, B))
    if most == 700:
        new = np.where(rng.random(B) < 0.9, np.minimum(new, 5), new)
    with Dev() as d:
        run(d, Case("lists", new, rng.integers(-1, adapters, B), adapters, 20, 72, 80, "bf16", "bf16", "f32", padding=3))


def test_requests_that_overlap_are_reported(device):
    """More than 64 requests whose starts fall: nothing is listed for them."""
    c = Case("overlap", [2] * 80, [0] * 80, 1, 8, 64, 32)
    c.starts[1:80:2] = 160
    with Dev() as d:
        args, more = c.put(d)
        log("lora of requests that overlap")
        native.lora(*args, **more)
        with pytest.raises(native.SlhipCacheError):
            native.synchronize()
        native.synchronize()
        assert (d.get(c.py, (c.T, c.N), np.float32) == -777.25).all()


@pytest.mark.parametrize("x,w,y", TYPES[:2])
def test_4096_requests(device, x, w, y):
    rng = rng_of("4096")
    new = rng.integers(0, 3, 4096)
    with Dev() as d:
        run(d, Case("4096", new, rng.integers(-1, 9, 4096), 9, 8, 40, 24, x, w, y, padding=5))


@pytest.mark.parametrize("x,w,y", [("bf16", "bf16", "bf16"), ("f32", "f16", "f32")])
@pytest.mark.parametrize("kw", [
    dict(in_place=True), dict(in_place=True, y_stride=101), dict(shift=1), dict(shift=1, x_stride=131, add_stride=97, y_stride=99, a_pad=3, b_pad=5),
    dict(x_stride=136, add_stride=104, y_stride=112, a_pad=8, b_pad=16)])
@pytest.mark.parametrize("most", [1, 90])
def test_strides_and_alignment(device, kw, most, x, w, y):
    rng = rng_of("strides", most)
    new = rng.integers(1, most + 1, 6)
    with Dev() as d:
        run(d, Case("strides", new, [0, 2, -1, 0, 1, 2], 3, 12, 128, 96, x, w, y, padding=3), **kw)


@pytest.mark.parametrize("y", ["f32", "bf16"])
def test_nothing_to_add(device, y):
    with Dev() as d:
        v = run(d, Case("null", [3, 2, 40], [0, -1, 1], 2, 16, 64, 80, y, "bf16", y, add=False))
        assert (v[3:5] == 0).all()


def test_no_adapters_at_all(device):
    """A set of no adapters: y is add, in place nothing is touched."""
    for in_place in (False, True):
        with Dev() as d:
            c = Case("none", [3, 70], [-1, -1], 1, 16, 64, 80, "bf16", "bf16", "bf16")
            args, more = c.put(d, in_place=in_place)
            args[5].adapters, args[5].a, args[5].b = 0, None, None
            log(f"lora of no adapters in_place={in_place}")
            native.lora(*args, **more)
            native.synchronize()
            c.check(d)


@pytest.mark.parametrize("x,w,y", TYPES[:4])
@pytest.mark.parametrize("most", [1, 80])
def test_unread_ranks_and_other_adapters(device, most, x, w, y):
    """What lies behind an adapter's ranks, and adapters that no request has, may be anything."""
    c = Case("unread", [most] * 4, [0, 2, 0, 2], 4, 21, 100, 90, x, w, y, ranks=[5, 21, 17, 3])
    nan = np.uint16(0x7FC0) if w == "bf16" else np.nan
    for ad in range(4):
        r = 0 if ad in (1, 3) else c.ranks[ad]
        c.a[ad, r:], c.b[ad, :, r:] = nan, nan
        c.va[ad, r:], c.vb[ad, :, r:] = 0, 0
    with Dev() as d:
        run(d, c)


@pytest.mark.parametrize("x,w,y", TYPES[:4])
def test_rows_that_are_not_finite_stay_alone(device, x, w, y):
    c = Case("inf", [40, 1, 1], [0, 1, 1], 2, 16, 64, 48, x, w, y)
    bad = {7: np.inf, 20: np.nan, 41: -np.inf}
    clean = c.expected()[0]
    for r, v in bad.items():
        c.vx[r, 3] = v
        c.x[r, 3] = oracle.to_bf16(np.float32([v]))[0] if x == "bf16" else v
    with Dev() as d:
        args, more = c.put(d)
        log(f"lora rows not finite {x}/{w}/{y}")
        native.lora(*args, **more)
        native.synchronize()
        got = values(d.get(c.py, (c.T, c.N), NP[y]), y)
    others = [t for t in range(c.T) if t not in bad]
    _, bound = step_ref.lora(np.nan_to_num(c.vx, nan=0, posinf=0, neginf=0), c.vadd, c.va, c.vb, c.starts, c.adapter, bf16_parts=True)
    assert (np.abs(got - clean)[others] <= step_ref.rounded_bound(clean, bound, y)[others]).all()
    assert not np.isfinite(got[list(bad)]).any()


def test_bad_adapters_and_requests_are_reported(device):
    for adapter, starts, error in (([0, 5, 1], None, IndexError), ([0, -2, 1], None, IndexError), ([0, 1, 1], [0, 3, 5, 90], native.SlhipCacheError),
                                   ([0, 1, 1], [-3, 3, 5, 6], native.SlhipCacheError)):
        c = Case("bad", [3, 2, 1], [0, 1, 1], 2, 8, 64, 32)
        c.adapter = np.int32(adapter)
        with Dev() as d:
            args, more = c.put(d)
            if starts:
                args[6].starts = d.put(np.int32(starts))
            log(f"lora bad adapter={adapter} starts={starts}")
            native.lora(*args, **more)
            with pytest.raises(error):
                native.synchronize()
            native.synchronize()
            if not starts:
                c.check(d)  # as -1
                continue
            got = d.get(c.py, (c.T, c.N), np.float32)
            y, bound = c.expected()
            rows = slice(0, 5) if starts[3] == 90 else slice(3, 6)
            assert (np.abs(got - y)[rows] <= step_ref.rounded_bound(y, bound, "f32")[rows]).all()
            left = slice(5, 6) if starts[3] == 90 else slice(0, 3)
            assert (got[left] == -777.25).all()


def test_captured_and_replayed_with_other_requests(device):
    """A captured step replays with other lengths and adapters; eager calls with a workspace of their own between replays."""
    rng = rng_of("graph")
    steps = [([1] * 9, [0, 1, 2, -1, 0, 0, 2, 1, 1]), ([3, 0, 0, 1, 2, 0, 1, 1, 0], [2, 1, 0, 0, 2, 2, -1, 1, 0]), ([9] + [0] * 8, [1] * 9)]
    st = native.Stream()
    with Dev() as d:
        c = Case("graph", *steps[0], 3, 16, 256, 192, "bf16", "bf16", "bf16", padding=2)
        args, more = c.put(d)
        other, other_more = Case("other", [30], [0], 1, 16, 256, 192, "bf16", "bf16", "bf16").put(d)
        eager = c.put(d)
        log("lora capture")
        g = native.Graph(st, lambda: native.lora(*args, **more, stream=st.handle))
        for rep in range(5):
            new, adapter = steps[rep % 3]
            c.starts, c.adapter = np.concatenate([[0], np.cumsum(new)]).astype(np.int32), np.int32(adapter)
            log(f"lora replay {rep}")
            for at in (args, eager[0]):
                for p, v in ((at[6].starts, c.starts), (at[6].adapter, c.adapter), (at[4], c.before)):
                    native.call("slhip_memcpy_h2d", p, v.ctypes.data, v.nbytes, st.handle)
            st.sync()
            native.lora(*other, **other_more, stream=st.handle)
            g.launch(st)
            native.lora(*eager[0], **eager[1], stream=st.handle)
            st.sync()
            got = d.get(args[4], (c.T, c.N), np.uint16)
            c.check(d, got)
            assert np.array_equal(got, d.get(eager[0][4], (c.T, c.N), np.uint16))
        del g


def test_captured_lists_of_tiles(device):
    """More than 64 requests in a captured step: it replays with other adapters, lengths and numbers of tiles."""
    rng = rng_of("graph of lists")
    B, T = 100, 260
    st = native.Stream()
    with Dev() as d:
        c = Case("lists", [1] * B, [0] * B, 40, 16, 128, 192, "bf16", "bf16", "bf16", padding=T - B)
        args, more = c.put(d)
        log("lora capture, 100 requests")
        g = native.Graph(st, lambda: native.lora(*args, **more, stream=st.handle))
        for rep in range(6):
            new = rng.integers(0, 4, B) if rep % 3 else np.full(B, 1)
            if rep == 4:
                new[:] = 0
                new[77] = T
            while new.sum() > T:
                new[rng.integers(0, B)] = 0
            adapter = rng.integers(-1, [40, 2, 1][rep % 3], B)
            c.starts, c.adapter = np.concatenate([[0], np.cumsum(new)]).astype(np.int32), adapter.astype(np.int32)
            for p, v in ((args[6].starts, c.starts), (args[6].adapter, c.adapter), (args[4], c.before)):
                native.call("slhip_memcpy_h2d", p, v.ctypes.data, v.nbytes, st.handle)
            st.sync()
            log(f"lora replay {rep}: {int(new.sum())} rows")
            g.launch(st)
            st.sync()
            c.check(d)
        del g


def test_two_streams_at_once(device):
    """Calls that overlap, each with its workspace; and the results do not change from call to call."""
    with Dev() as d:
        cases = [Case(f"s{i}", [60, 1, 30], [0, 1, 0], 2, 32, 512, 640, "f32", "bf16", "f32") for i in range(2)]
        calls = [c.put(d) for c in cases]
        streams = [native.Stream(), native.Stream()]
        native.synchronize()
        log("lora on two streams")
        for _ in range(20):
            for st, (args, more) in zip(streams, calls):
                native.lora(*args, **more, stream=st.handle)
        for st in streams:
            st.sync()
        first = [d.get(c.py, (c.T, c.N), np.float32) for c in cases]
        for c, got in zip(cases, first):
            c.check(d, got)
        native.lora(*calls[0][0], **calls[0][1])
        native.synchronize()
        assert np.array_equal(first[0], d.get(cases[0].py, (cases[0].T, cases[0].N), np.float32))


def test_a_long_prompt(device):
    """Rows over many tiles and ranges of K; only a sample of them is compared."""
    T, K, N, R = 2100, 2048, 1030, 16
    c = Case("long", [T - 100, 99], [1, 0], 2, R, K, N, "bf16", "bf16", "bf16", padding=1)
    with Dev() as d:
        args, more = c.put(d)
        log(f"lora T={T}")
        native.lora(*args, **more)
        native.synchronize()
        c.check(d)


@pytest.mark.parametrize("requests", [1, 3, 70])
def test_many_rows_and_columns(device, requests):
    """So many column steps that thread blocks take turns; a sample of the rows is compared, in every column."""
    rng = rng_of("turns", requests)
    T, K, N, R, padding = 4190, 64, 12540, 16, 6
    cuts = np.sort(rng.choice(np.arange(1, T - padding), requests - 1, replace=False))
    starts = np.concatenate([[0], cuts, [T - padding]]).astype(np.int32)
    adapter = rng.integers(0, 2, requests).astype(np.int32)
    x, vx = held(rng.standard_normal((T, K)), "bf16")
    a, va = held(rng.standard_normal((2, R, K)) / np.sqrt(K), "bf16")
    b, vb = held(rng.standard_normal((2, N, R)) / np.sqrt(R), "bf16")
    add = oracle.to_bf16(rng.standard_normal((T, N), dtype=np.float32))
    with Dev() as d:
        at = d.put(add)
        size = native.lora_work_bytes(T, R)
        log(f"lora T={T} N={N} requests={requests}")
        native.lora("bf16", "bf16", d.put(x), at, at, native.lora_set("bf16", d.put(a), d.put(b), 2, R, K, N),
                    native.lora_rows(requests, T, d.put(starts), d.put(adapter)), work=d.empty(size), work_bytes=size)
        native.synchronize()
        got = d.get(at, (T, N), np.uint16)
    assert np.array_equal(got[T - padding:], add[T - padding:])
    rows = np.unique(np.concatenate([rng.integers(0, T - padding, 150), np.arange(T - padding - 33, T - padding), cuts, starts[:-1]]))
    which = np.searchsorted(starts, rows, side="right") - 1
    y, bound = step_ref.lora(vx[rows], values(add[rows], "bf16"), va, vb, np.arange(len(rows) + 1), adapter[which], bf16_parts=True)
    off = np.abs(values(got[rows], "bf16") - y)
    assert np.all(off <= step_ref.rounded_bound(y, bound, "bf16"))
