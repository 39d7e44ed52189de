"""GPU parity of draft verification (slhip_draft_verify) against the 64-bit statement of tests/step_ref.py: tokens and counts are equal, the
random numbers being chosen (before any run) so that no choice of the statement is nearer than 2^-20 to another; the
logarithms within the bound derived there."""
import numpy as np
import pytest

import oracle
from sharplight_amd import native
from tests import step_ref
from tests.devutil import Dev, log
from tests.test_gpu_lora import NP, SIZE, held, rng_of, wide

pytestmark = pytest.mark.gpu

NEAR = 2.0 ** -20


class Case:
    def __init__(self, name, new, V, dtype="f32", drawn=True, tau=None, tau_q=None, mask=0, padding=0, extra=0, good=0.6, size=2.5, settle=True):
        rng = rng_of(name, len(new), V, dtype, drawn)
        self.rng, self.new, self.V, self.dtype = rng, list(new), V, dtype
        self.starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        B, T = len(new), int(self.starts[-1]) + padding
        self.T, self.stride = T, max(list(new) + [1]) + extra
        z = rng.standard_normal((T, V)) * size
        near = z + rng.standard_normal((T, V)) * 0.5
        if mask:
            z[rng.random((T, V)) < mask] = -np.inf
            z[np.arange(T), rng.integers(0, V, T)] = 1.0  # one is left in any case
        self.target, self.z = held(z, dtype)
        self.draft, self.q = held(near, dtype) if drawn else (None, None)
        self.tau = None if tau is None else np.float32(rng.choice(tau, B))
        self.tau_q = None if tau_q is None else np.float32(rng.choice(tau_q, B))
        likely = rng.random(T) < good
        self.ids = np.where(likely, z.argmax(-1), rng.integers(0, V, T)).astype(np.int32)
        self.ids = np.roll(self.ids, 1)
        self.past = rng.integers(0, 5000, B).astype(np.int32)
        self.accept, self.sample = (rng.random(n).astype(np.float32) for n in (T, B))
        if settle:
            self.settle()

    def statement(self, **kw):
        a = dict(target=self.z, draft=self.q, starts=self.starts, ids=self.ids, accept=self.accept.astype(np.float64), sample=self.sample.astype(np.float64),
                 stride=self.stride, tau=self.tau, tau_q=self.tau_q, past=self.past)
        a.update(kw)
        return step_ref.verify(**a)

    def settle(self):
        """New random numbers for requests whose choices are too near to another, until none is left."""
        for i in range(len(self.new)):
            s = slice(self.starts[i], self.starts[i + 1])
            for _ in range(50):
                one = self.statement(starts=np.int32([self.starts[i], self.starts[i + 1]]), sample=self.sample[i:i + 1].astype(np.float64), past=self.past[i:i + 1],
                                     tau=None if self.tau is None else self.tau[i:i + 1], tau_q=None if self.tau_q is None else self.tau_q[i:i + 1])
                if one[5] > NEAR:
                    break
                self.accept[s] = self.rng.random(s.stop - s.start)
                self.sample[i] = self.rng.random()
            else:
                raise AssertionError("no random numbers that settle the choices")

    def put(self, d, target_stride=None, draft_stride=None, shift=0, logp=True, lengths=True):
        nan = np.float32(np.nan) if self.dtype == "f32" else np.uint16(0x7FC0)
        zs, qs = target_stride or self.V, draft_stride or self.V
        pt = d.put(wide(self.target, zs, nan), pad_bytes=shift * SIZE[self.dtype])
        pd = None if self.draft is None else d.put(wide(self.draft, qs, nan), pad_bytes=shift * SIZE[self.dtype])
        B = len(self.new)
        opt = lambda v: None if v is None else d.put(v)  # noqa: E731
        self.at = {k: d.empty(4 * max(n, 1)) for k, n in (("out", B * self.stride), ("n_out", B), ("kept", B), ("dropped", B), ("logp", B * self.stride))}
        dr = native.drafts(B, self.T, self.V, d.put(self.starts), d.put(self.ids), d.put(self.accept), d.put(self.sample), self.at["out"], self.stride,
                           self.at["n_out"], temperature=opt(self.tau), draft_temperature=opt(self.tau_q), past=d.put(self.past) if lengths else None,
                           kept=self.at["kept"] if lengths else None, dropped=self.at["dropped"] if lengths else None, logp=self.at["logp"] if logp else None)
        size = native.draft_verify_work_bytes(B, self.T, self.V)
        return (self.dtype, pt, pd, dr), dict(target_stride=zs, draft_stride=qs, work=d.empty(max(size, 16)), work_bytes=size)

    def check(self, d, logp=True, lengths=True, want=None):
        B = len(self.new)
        out, n_out, kept, dropped, lp, _ = want or self.statement()
        got = {k: d.get(self.at[k], (B, self.stride) if k in ("out", "logp") else (B,), np.float32 if k == "logp" else np.int32) for k in self.at}
        assert np.array_equal(got["n_out"], n_out), np.nonzero(got["n_out"] != n_out)[0][:5]
        assert np.array_equal(got["out"], out), np.argwhere(got["out"] != out)[:5]
        if lengths:
            assert np.array_equal(got["kept"], kept) and np.array_equal(got["dropped"], dropped)
        else:
            assert (got["kept"] == np.int32(-0x54545455)).all()
        if logp:
            for i in range(B):
                for j in range(self.stride):
                    if j >= n_out[i]:
                        assert got["logp"][i, j] == 0
                    elif np.isnan(lp[i, j]):
                        assert np.isnan(got["logp"][i, j])
                    else:
                        t = 1.0 if self.tau is None else float(self.tau[i])
                        bound = step_ref.logp_bound(self.z[self.starts[i] + j], t, lp[i, j])
                        assert abs(got["logp"][i, j] - lp[i, j]) <= bound, (i, j, got["logp"][i, j], lp[i, j], bound)
        return got


def run(d, c, **kw):
    args, more = c.put(d, **kw)
    log(f"draft_verify B={len(c.new)} T={c.T} V={c.V} {c.dtype} draft={c.draft is not None} {kw}")
    native.draft_verify(*args, **more)
    native.synchronize()
    return c.check(d, logp=kw.get("logp", True), lengths=kw.get("lengths", True))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("drawn", [True, False])
@pytest.mark.parametrize("new,V", [([1], 1), ([3], 2), ([5], 7), ([4], 255), ([6], 4095), ([6], 4096), ([6], 4097), ([2, 5, 1], 8191), ([17], 1000), ([3, 4], 32001)])
def test_sizes(device, new, V, dtype, drawn):
    with Dev() as d:
        run(d, Case("sizes", new, V, dtype, drawn))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("drawn,tau,tau_q,mask", [
    (True, [0.0, 0.5, 1.0, 1.7], None, 0), (True, [0.7, 1.0], [0.0, 0.5, 2.0], 0), (False, [-1.0, 0.3, 1.0], None, 0.9), (True, [1.0], None, 0.5),
    (True, [0.0], None, 0), (False, [1.0, 3.0], [0.0], 0.99), (True, [0.01, 100.0], [1.0], 0)])
def test_temperatures_and_masks(device, drawn, tau, tau_q, mask, dtype):
    rng = rng_of("temperatures", tau)
    new = rng.integers(0, 6, 40)
    with Dev() as d:
        run(d, Case("temperatures", new, 1234, dtype, drawn, tau, tau_q, mask, padding=3, extra=2))


@pytest.mark.parametrize("B", [65, 300, 4200])
def test_many_requests(device, B):
    rng = rng_of("many", B)
    new = rng.integers(0, 4, B)
    with Dev() as d:
        run(d, Case("many", new, 100, "f32", True, [0.0, 1.0], padding=9))


@pytest.mark.parametrize("new", [[40], [1, 33, 8, 16, 9]])
def test_long_drafts(device, new):
    """More rows than a pass over them takes, mostly accepted."""
    with Dev() as d:
        run(d, Case("long", new, 300, "f32", True, good=1.0, size=6.0))
        run(d, Case("long greedy", new, 300, "f32", False, [0.0], good=1.0))


@pytest.mark.parametrize("kw", [dict(target_stride=1003, draft_stride=1010), dict(shift=1), dict(shift=1, target_stride=1001), dict(logp=False, lengths=False),
                                dict(target_stride=1008, draft_stride=1024)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides_and_alignment(device, kw, dtype):
    with Dev() as d:
        run(d, Case("strides", [3, 1, 5], 999, dtype, True, [0.0, 1.0]), **kw)


def test_a_large_vocabulary(device):
    with Dev() as d:
        run(d, Case("large", [5, 2, 1], 151936, "f32", True, size=2.0))
        run(d, Case("large bf16", [5, 2, 1], 262144, "bf16", False, [0.0, 0.8], size=2.0))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_ties_go_to_the_lowest(device, dtype):
    c = Case("ties", [4, 1, 3], 9000, dtype, False, [0.0])
    c.z = np.round(c.z)  # many equal largest logits
    c.target, c.z = held(c.z, dtype)
    c.ids = np.roll(np.where(np.arange(c.T) % 3 < 2, c.z.argmax(-1), 8999 - c.z[:, ::-1].argmax(-1)), 1).astype(np.int32)
    with Dev() as d:
        run(d, c)


def test_random_numbers_at_the_ends(device):
    """0, the largest below 1, and 1 and NaN, which no generator gives: the first and the last token with a weight."""
    c = Case("ends", [1, 1, 1, 1, 1], 5000, "f32", False, mask=0.5, settle=False)
    c.z[:, :3], c.z[:, 4900:] = -np.inf, -np.inf
    c.target = c.z.astype(np.float32)
    c.sample = np.float32([0.0, 1 - 2.0 ** -24, 1.0, np.nan, 2.0])
    first = [int(np.nonzero(r > -np.inf)[0][0]) for r in c.z]
    last = [int(np.nonzero(r > -np.inf)[0][-1]) for r in c.z]
    with Dev() as d:
        args, more = c.put(d)
        log("draft_verify samples at the ends")
        native.draft_verify(*args, **more)
        native.synchronize()
        out = d.get(c.at["out"], (5, 1), np.int32)[:, 0]
    assert out[0] == first[0] and out[2] == last[2] and out[3] == first[3] and out[4] == last[4]
    p = step_ref.probabilities(c.z[1], 1.0)
    assert p[out[1]:].sum() > 2.0 ** -26 and p[out[1] + 1:].sum() < 2.0 ** -22


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_equal_probabilities_accept_all(device, dtype):
    """A draft model that is the target: no random number below 1 refuses anything."""
    c = Case("equal", [6, 6, 6], 3000, dtype, True, settle=False)
    c.draft, c.q = c.target, c.z
    c.accept[:] = 1 - 2.0 ** -24
    c.sample[:] = 0.5
    with Dev() as d:
        args, more = c.put(d)
        log("draft_verify equal probabilities")
        native.draft_verify(*args, **more)
        native.synchronize()
        out, n = d.get(c.at["out"], (3, 6), np.int32), d.get(c.at["n_out"], (3,), np.int32)
    assert (n == 6).all()
    for i in range(3):
        assert np.array_equal(out[i, :5], c.ids[6 * i + 1:6 * i + 6])


def test_a_refused_draft_of_equal_probabilities_draws_from_the_target(device):
    """accept = 1 refuses it, nothing is left of p - q: the weights are p."""
    c = Case("left", [2, 2], 9000, "f32", True, settle=False)
    c.draft, c.q = c.target, c.z
    c.accept[:] = 1.0
    c.sample[:] = [0.3, 0.8]
    with Dev() as d:
        args, more = c.put(d)
        log("draft_verify nothing left")
        native.draft_verify(*args, **more)
        native.synchronize()
        c.check(d)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("drawn", [True, False])
def test_rows_that_cannot_be_used(device, drawn, dtype):
    """NaN, +inf and nothing above -inf in the target's rows and in the draft's; a NaN temperature."""
    c = Case("unusable", [3] * 9, 5000, dtype, drawn, [1.0, 0.0], good=1.0, size=5.0, settle=False)
    c.tau[:] = [1.0, 1.0, 1.0, 0.0, 0.0, 1.0, 1.0, np.nan, 1.0]
    c.accept[:] = 0.01
    for row, v in ((0, np.nan), (4, np.inf), (8, -np.inf), (9, np.nan), (13, -np.inf)):
        c.z[row, 4999 if np.isnan(v) or v > 0 else slice(None)] = v
    c.target, c.z = held(c.z, dtype)
    if drawn:
        c.q[15, 17], c.q[19, :] = np.nan, -np.inf
        c.draft, c.q = held(c.q, dtype)
    want = c.statement()
    assert want[5] > NEAR
    with Dev() as d:
        args, more = c.put(d)
        log(f"draft_verify unusable rows drawn={drawn} {dtype}")
        native.draft_verify(*args, **more)
        native.synchronize()
        got = c.check(d, want=want)
    assert got["out"][0, 0] == -1 and got["out"][1, 1] == -1 and got["out"][2, 2] == -1 and got["out"][7, 0] == -1


def test_masks_of_the_lowest_number(device):
    c = Case("lowest", [3, 1, 2], 6000, "f32", True, [0.5, 1.0], mask=0.9)
    c.z[c.z == -np.inf] = np.finfo(np.float32).min
    c.target = c.z.astype(np.float32)
    with Dev() as d:
        run(d, c)
    c = Case("all lowest", [1], 6000, "f32", False)  # all alike: a finite row
    c.z[:] = np.finfo(np.float32).min
    c.target = c.z.astype(np.float32)
    c.settle()
    with Dev() as d:
        run(d, c)


def test_bad_drafts_and_requests_are_reported(device):
    for ids, stride, starts, error in ((777, 3, None, IndexError), (-1, 3, None, IndexError), (None, 2, None, native.SlhipCacheError),
                                       (None, 3, [0, 2, 4, 60], native.SlhipCacheError), (None, 3, [0, 2, 1, 4], native.SlhipCacheError)):
        c = Case("bad", [3, 2, 1], 700, "f32", True, settle=False)
        c.accept[:] = 0.0
        c.stride = stride
        if starts:
            c.starts = np.int32(starts)
        if ids is not None:
            c.ids[1] = ids
        with Dev() as d:
            args, more = c.put(d)
            log(f"draft_verify bad ids={ids} stride={stride} starts={starts}")
            native.draft_verify(*args, **more)
            with pytest.raises(error):
                native.synchronize()
            native.synchronize()
            out, n = d.get(c.at["out"], (3, stride), np.int32), d.get(c.at["n_out"], (3,), np.int32)
        if ids is not None:
            assert n[0] == 1 and 0 <= out[0, 0] < 700 and n[1] == 2 and n[2] == 1
        elif stride == 2:
            assert n.tolist() == [0, 2, 1] and (out[0] == -1).all()
        elif starts[3] == 60:
            assert n.tolist()[2] == 0 and (out[2] == -1).all() and n[0] == 2
        else:
            assert n[1] == 0 and (out[1] == -1).all()


def test_a_draft_behind_a_refused_one_is_not_looked_at(device):
    c = Case("behind", [4], 700, "f32", False, settle=False)
    c.accept[:] = 1.0  # the first one is refused
    c.ids[2] = 12345
    with Dev() as d:
        args, more = c.put(d)
        log("draft_verify behind a refused draft")
        native.draft_verify(*args, **more)
        native.synchronize()
        assert d.get(c.at["n_out"], (1,), np.int32)[0] == 1


def test_no_rows(device):
    with Dev() as d:
        c = Case("nothing", [0, 0], 100, "f32", True, padding=2)
        got = run(d, c)
        assert (got["n_out"] == 0).all() and (got["out"] == -1).all() and np.array_equal(got["kept"], c.past)
        c.T = 0
        args, more = c.put(d)
        log("draft_verify T=0")
        native.draft_verify(*args, **more)
        native.synchronize()
        c.check(d)


def test_captured_and_replayed(device):
    """A captured call replays with other rows, drafts, random numbers and temperatures, eager work between the replays."""
    st = native.Stream()
    with Dev() as d:
        cases = [Case(f"replay{i}", new, 5000, "bf16", True, [0.0, 1.0], padding=12 - sum(new), extra=8 - max(new)) for i, new in
                 enumerate(([5, 1, 3], [1, 1, 1], [0, 8, 4]))]
        c = cases[0]
        args, more = c.put(d)
        dr = args[3]
        log("draft_verify capture")
        g = native.Graph(st, lambda: native.draft_verify(*args, **more, stream=st.handle))
        eager = Case("eager", [4, 4], 5000, "bf16", True)
        eargs, emore = eager.put(d)
        for rep in range(6):
            n = cases[rep % 3]
            n.at = c.at
            for p, v in ((args[1], n.target), (args[2], n.draft), (dr.starts, n.starts), (dr.ids, n.ids), (dr.accept, n.accept), (dr.sample, n.sample),
                         (dr.temperature, n.tau), (dr.past, n.past)):
                native.call("slhip_memcpy_h2d", p, v.ctypes.data, v.nbytes, st.handle)
            native.draft_verify(*eargs, **emore, stream=st.handle)
            st.sync()
            log(f"draft_verify replay {rep}")
            g.launch(st)
            st.sync()
            n.check(d)
            eager.check(d)
        del g


@pytest.mark.parametrize("B", [5, 700])
@pytest.mark.parametrize("drawn", [True, False])
def test_lengths_in_place(device, drawn, B):
    """kept is past: a step's lengths become the next one's; a request that does not fit keeps its own."""
    c = Case("lengths", ([3, 1, 4, 2, 3] * 140)[:B], 300, "f32", drawn, extra=0)
    with Dev() as d:
        (dt, target, draft, dr), more = c.put(d)
        log(f"draft_verify kept = past B={B} drawn={drawn}")
        dr.kept = dr.past
        want = c.statement()
        native.draft_verify(dt, target, draft, dr, **more)
        native.synchronize()
        assert np.array_equal(d.get(dr.past, (B,), np.int32), want[2]) and np.array_equal(d.get(c.at["dropped"], (B,), np.int32), want[3])
        now = want[2].astype(np.int32)
        dr.out_stride = 3  # the requests of four rows do not fit
        native.draft_verify(dt, target, draft, dr, **more)
        with pytest.raises(native.SlhipCacheError, match="does not fit"):
            native.synchronize()
        n_out = np.where(np.diff(c.starts) > 3, 0, want[1])
        assert np.array_equal(d.get(dr.past, (B,), np.int32), now + n_out)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_most_requests_times_chunks(device, dtype):
    """More chunks of all requests than one dimension of a launch takes; few of the requests have rows, the last one among them."""
    B, V = 40000, 1 << 20
    new = np.zeros(B, int)
    new[[0, 20011, B - 2, B - 1]] = [2, 1, 2, 2]
    c = Case("most", new.tolist(), V, dtype, True, good=0.0, size=12.0)
    with Dev() as d:
        run(d, c)


def test_one_token_in_the_vocabulary(device):
    for drawn in (True, False):
        with Dev() as d:
            run(d, Case("single", [1, 3, 2], 1, "f32", drawn))


def test_two_streams_at_once(device):
    with Dev() as d:
        cases = [Case(f"stream{i}", [4, 2, 5], 40000, "f32", True) for i in range(2)]
        calls = [c.put(d) for c in cases]
        streams = [native.Stream(), native.Stream()]
        native.synchronize()
        log("draft_verify on two streams")
        for _ in range(20):
            for st, (args, more) in zip(streams, calls):
                native.draft_verify(*args, **more, stream=st.handle)
        for st in streams:
            st.sync()
        for c in cases:
            c.check(d)
