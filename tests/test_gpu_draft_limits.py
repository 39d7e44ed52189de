"""Draft verification where its numbers are at their ends: random numbers of 0 and 1 beside tokens far below the others, drafts that hold nearly
all of p, sums of many small terms, the largest temperature, rows and temperatures that cannot be used. The 64-bit statement is
tests/step_ref.py's."""
import numpy as np
import pytest

from sharplight_amd import native
from tests import step_ref
from tests.devutil import Dev, log
from tests.test_gpu_draft import NEAR, Case
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
        assert p[x] > 0, (i, x, p[x], logp[i, 0])
        weighty = np.nonzero(p > 2.0 ** -100 * p.max())[0]
        if i in (0, 2, 4):
            assert x <= weighty[0]
        else:
            assert x >= weighty[-1]


# ---- drafts that hold nearly all of p ------------------------------------------------------------------------------

def _others(c, at, places, weights):
    """Rows of one draft at `at` (logit 0) and others of the given weights; all else is masked. Returns the places and what they weigh."""
    z = np.full((c.T, c.V), -np.inf)
    z[:, at] = 0.0
    z[:, places] = np.log(weights)
    c.target, c.z = held(z, c.dtype)
    c.ids[:] = at
    c.accept[:] = 1 - 2.0 ** -24
    order = np.sort(places)
    return order, np.exp(c.z[0, order])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("by_temperature", [False, True])
@pytest.mark.parametrize("at,places", [(5, [4, 6, 7]), (5, [0, 1, 2, 3, 4, 6, 7]), (4101, [4100, 4102, 4103]), (9, [8, 10, 11, 2060, 2061])])
def test_a_refused_draft_of_nearly_all_is_not_drawn(device, at, places, by_temperature, dtype):
    """The others weigh less than half of 2^-24 each: all of them vanish in f32 beside the draft's 1."""
    c = Case("nearly all", [2] * len(places), 5000, dtype, by_temperature, [1.0], [0.0], settle=False)
    order, w = _others(c, at, places, np.full(len(places), 0.45 * 2.0 ** -24) if len(places) > 5 else np.full(len(places), 0.8 * 2.0 ** -24))
    share = np.cumsum(w) / w.sum()
    c.sample = np.float32(share - 0.5 * w / w.sum())  # the middle of each one's part
    with Dev() as d:
        out, n, logp = _call(d, c, f"a draft of nearly all at {at} {dtype}")
    assert (n == 1).all() and np.array_equal(out[:, 0], order), out[:, 0]
    want = np.log(step_ref.probabilities(c.z[0], 1.0)[order])
    assert np.all(np.abs(logp[:, 0] - want) <= [step_ref.logp_bound(c.z[0], 1.0, v) for v in want])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("by_temperature", [False, True])
@pytest.mark.parametrize("at,total", [(5, 2.0 ** -20), (4999, 2.0 ** -17), (4097, 2.0 ** -14), (100, 2.0 ** -10)])
def test_what_is_left_of_a_chunk_is_summed_without_the_draft(device, at, total, by_temperature, dtype):
    """p(x) = 1 - total, the rest over x's chunk and the others: every one of them is drawn by the middle of its part, whose halves are 2^-9 of
    the rest or more."""
    V, n = 12000, 100
    c = Case("left", [2] * n, V, dtype, by_temperature, [1.0], [0.0], settle=False)
    chunk = 4096 if dtype == "f32" else 8192
    inside = np.arange(at // chunk * chunk, min((at // chunk + 1) * chunk, V))
    inside = inside[inside != at]
    rest = np.setdiff1d(np.arange(V), np.append(inside, at))
    places = np.concatenate([c.rng.choice(inside, 80, replace=False), c.rng.choice(rest, 20, replace=False)])
    order, w = _others(c, at, places, total / n * (0.7 + 0.6 * c.rng.random(n)))
    share = np.cumsum(w) / w.sum()
    c.sample = np.float32(share - 0.5 * w / w.sum())
    assert (0.5 * w / w.sum()).min() > 2.0 ** -9
    with Dev() as d:
        out, got, _ = _call(d, c, f"what is left beside {at} {total} {dtype}")
    assert (got == 1).all() and np.array_equal(out[:, 0], order), np.nonzero(out[:, 0] != order)[0]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_what_is_left_in_a_large_vocabulary(device, dtype):
    """Drafts in chunks behind the first 64."""
    V, n = 600000, 40
    c = Case("left, large", [2] * n, V, dtype, False, settle=False)
    at = 590001
    places = np.concatenate([np.arange(at - 20, at), np.arange(at + 1, at + 11), c.rng.choice(500000, 10, replace=False)])
    order, w = _others(c, at, places, 2.0 ** -22 / n * (0.7 + 0.6 * c.rng.random(n)))
    c.sample = np.float32(np.cumsum(w) / w.sum() - 0.5 * w / w.sum())
    with Dev() as d:
        out, got, _ = _call(d, c, f"what is left of a large vocabulary {dtype}")
    assert (got == 1).all() and np.array_equal(out[:, 0], order)


# ---- random numbers next to a border -------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,V,B", [("f32", 151936, 24), ("bf16", 50257, 48), ("f32", 1200, 48), ("bf16", 20000, 48), ("f32", 300000, 8)])
@pytest.mark.parametrize("kind", ["no draft", "drawn", "chosen", "chosen by a temperature", "all accepted"])
@pytest.mark.parametrize("tau", [1.0, 0.6])
def test_random_numbers_next_to_a_border(device, tau, kind, dtype, V, B):
    """A row has as many borders as tokens, so among many draws some random number lies next to one. Here each is the f32 number that lies nearest to
    one of them, 2^-36 / R of the sum or more away from it, of weights that sum to R: terms that are off by 2^-39, above and below the fraction, put a border
    off by 2^-38 at most, and where they are differences p - q by 2^-37 / R. What is drawn is the statement's token, and no other."""
    drawn = kind in ("drawn", "all accepted", "chosen by a temperature")
    c = Case("border" + kind, [1 if kind == "no draft" else 2] * B, V, dtype, drawn, [tau], [0.0] if kind == "chosen by a temperature" else [tau], settle=False)
    c.z += 6.0 * (c.rng.random(c.z.shape) < 8.0 / V)
    c.target, c.z = held(c.z, dtype)
    c.accept[:] = 0.0 if kind == "all accepted" else 1 - 2.0 ** -24
    want, near = np.zeros(B, int), np.zeros(B)
    t = float(np.float32(tau))
    for i in range(B):
        row = c.starts[i]
        if kind == "all accepted":
            c.ids[row + 1] = c.z[row].argmax()
            row += 1
        w = step_ref.probabilities(c.z[row], t)
        if kind == "drawn":
            q = step_ref.probabilities(c.q[row], t)
            c.ids[row + 1] = (q - w).argmax()
            w = np.maximum(w - q, 0.0)
        elif kind.startswith("chosen"):
            c.ids[row + 1] = c.rng.choice(V, p=w)
            w[c.ids[row + 1]] = 0.0
        least = 2.0 ** -36 / w.sum()
        share = np.cumsum(w.astype(np.longdouble))
        share /= share[-1]
        u = np.float32(share[:-1])  # the nearest f32 numbers
        off = np.abs(u - share[:-1]).astype(np.float64)
        off[(off < least) | (u >= 1) | (w[1:] == 0)] = 1.0
        v = off.argmin()
        c.sample[i], near[i] = u[v], off[v]
        want[i] = np.searchsorted(share, np.longdouble(u[v]), side="right")
    if V > 10000:
        assert np.median(near) < 2.0 ** -28
    with Dev() as d:
        out, n, _ = _call(d, c, f"next to a border {kind} {dtype} V={V} tau={tau}")
    place = 1 if kind == "all accepted" else 0
    assert (n == place + 1).all() and np.array_equal(out[:, place], want), np.nonzero(out[:, place] != want)[0]


# ---- sums ----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,far,step", [("f32", 1024, 4), ("bf16", 2048, 8)])
def test_small_terms_beside_a_large_one(device, dtype, far, step):
    """All logits that one thread adds are just below half a unit of its first one: the row's sum stays within the bound that 16 f32 terms give."""
    c = Case("small terms", [1], 20000, dtype, False, settle=False)
    c.z[:] = -np.inf
    for j in range(4):
        c.z[:, far * j:far * j + step] = -16.75  # e^-16.75 = 0.89 * 2^-24
    c.z[:, 0] = 0.0
    c.target, c.z = held(c.z, dtype)
    c.sample[:] = 0.0
    with Dev() as d:
        out, n, logp = _call(d, c, f"small terms {dtype}")
    want = np.log(step_ref.probabilities(c.z[0], 1.0)[0])
    assert n[0] == 1 and out[0, 0] == 0
    assert abs(logp[0, 0] - want) <= step_ref.logp_bound(c.z[0], 1.0, want), (logp[0, 0], want)


@pytest.mark.parametrize("tau", [2.0 ** 40, 2.0 ** 60, 2.0 ** 38, 2.0 ** 20, 2.0 ** -20, 2.0 ** -40, 2.0 ** -60])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_temperatures_at_the_ends(device, tau, dtype):
    """One token, and 4000 of the same chunk that weigh as much together: an exponent's error counts half."""
    V = 4001
    c = Case("temperatures", [1], V, dtype, False, [tau], settle=False)
    heat = min(max(tau, 2.0 ** -40), 2.0 ** 40)
    c.z[:] = np.log(1 / 4000) * heat
    c.z[:, 77] = 0.0
    c.target, c.z = held(c.z, dtype)
    p = step_ref.probabilities(c.z[0], tau)
    c.sample[:] = p[:77].sum() + 0.5 * p[77]
    with Dev() as d:
        out, n, logp = _call(d, c, f"temperature {tau} {dtype}")
    want = np.log(p[77])
    assert n[0] == 1 and out[0, 0] == 77
    assert abs(logp[0, 0] - want) <= step_ref.logp_bound(c.z[0], tau, want), (logp[0, 0], want)


# ---- rows, drafts and temperatures that cannot be used -------------------------------------------------------------

@pytest.mark.parametrize("drawn", [True, False])
@pytest.mark.parametrize("why", ["nan", "inf", "masked", "temperature"])
@pytest.mark.parametrize("x", [5000, -1, 1 << 30])
def test_a_bad_draft_of_a_row_that_cannot_be_used_is_reported(device, x, why, drawn):
    c = Case("bad both", [1, 3, 2], 5000, "f32", drawn, [1.0], settle=False)
    c.ids[2] = x  # the draft of request 1's first row
    if why == "temperature":
        c.tau[1] = np.nan
    else:
        c.z[1, 17 if why != "masked" else slice(None)] = {"nan": np.nan, "inf": np.inf, "masked": -np.inf}[why]
    c.target, c.z = held(c.z, "f32")
    with Dev() as d:
        args, more = c.put(d)
        log(f"draft_verify bad draft {x} of a row that cannot be used: {why} drawn={drawn}")
        native.draft_verify(*args, **more)
        with pytest.raises(IndexError, match="number 0 of request 1"):
            native.synchronize()
        native.synchronize()
        out, n = d.get(c.at["out"], (3, 3), np.int32), d.get(c.at["n_out"], (3,), np.int32)
    assert n[1] == 1 and (out[1] == -1).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [1, 7, 5000, 8191])
@pytest.mark.parametrize("behind", [0, 1, 8])
def test_a_chosen_draft_behind_the_vocabulary(device, behind, V, dtype):
    """In what would be the last chunk: refused and reported, and what lies behind the row's logits (NaN, or nothing) is not looked at."""
    c = Case("behind", [2, 2, 2], V, dtype, False, [1.0, 0.6], settle=False)
    c.ids[1::2] = V + behind
    c.sample[:] = [0.2, 0.5, 0.9]
    want = c.statement()
    assert want[5] > NEAR and (want[1] == 1).all()
    for stride in (V, V + 24):
        with Dev() as d:
            args, more = c.put(d, target_stride=stride)
            log(f"draft_verify chosen draft {V + behind} of {V}, stride {stride} {dtype}")
            native.draft_verify(*args, **more)
            with pytest.raises(IndexError, match="number 0 of request"):
                native.synchronize()
            native.synchronize()
            c.check(d, want=want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_draft_temperature_that_is_not_a_number(device, dtype):
    """Counts as draft logits that cannot be used: the draft is refused, the token drawn from p. Without draft logits none is looked at."""
    c = Case("nan draft temperature", [3, 2, 1], 5000, dtype, True, [1.0], [1.0], good=1.0, size=5.0, settle=False)
    c.tau_q[:2] = np.nan
    c.accept[:], c.sample[:] = 0.0, 0.6
    want = c.statement()
    assert want[5] > NEAR and want[1].tolist() == [1, 1, 1]
    with Dev() as d:
        args, more = c.put(d)
        log(f"draft_verify NaN draft temperature {dtype}")
        native.draft_verify(*args, **more)
        native.synchronize()
        c.check(d, want=want)
        c.q, c.draft = None, None
        want = c.statement(tau_q=None)
        assert want[5] > NEAR and want[1].tolist() == [3, 2, 1]
        args, more = c.put(d)
        log(f"draft_verify NaN draft temperature, no draft logits {dtype}")
        native.draft_verify(*args, **more)
        native.synchronize()
        c.check(d, want=want)


# ---- lengths -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("drawn", [True, False])
def test_requests_of_too_many_rows_give_their_blocks_back(device, drawn):
    """A request with more rows than out_stride gets no token and drops all of its rows: the trim behind takes all their blocks back."""
    B, bs, bps = 4, 16, 6
    new, past = [40, 3, 33, 1], np.int32([7, 16, 0, 31])
    c = Case("too many rows", new, 300, "f32", drawn, settle=False)
    c.stride, c.past = 3, past
    pages = np.full((B, bps), -1, np.int32)
    ids = iter(range(100))
    for i in range(B):
        for j in range(-(-int(past[i]) // bs)):
            pages[i, j] = next(ids)
    free = np.int32([next(ids) for _ in range(12)])
    with Dev() as d:
        pp, pf, n, count, starts = d.put(pages), d.put(free), d.put(np.int32([12])), d.put(np.int32(new)), d.empty(4 * (B + 1))
        args, more = c.put(d)
        dr = args[3]
        log(f"advance, draft_verify of too many rows, trim; drawn={drawn}")
        native.kv_pages_advance(native.kv_pages(B, dr.past, count, pp, B, bps, bs, pf, 12, n, n, c.T, starts))
        native.draft_verify(*args, **more)
        native.kv_pages_trim(native.kv_pages(B, dr.kept, dr.dropped, pp, B, bps, bs, pf, 12, n, n))
        with pytest.raises(native.SlhipCacheError, match="does not fit"):
            native.synchronize()
        native.synchronize()
        n_out, kept, dropped = (d.get(c.at[k], (B,), np.int32) for k in ("n_out", "kept", "dropped"))
        assert n_out[0] == n_out[2] == 0 and n_out[3] == 1
        assert np.array_equal(kept, past + n_out) and np.array_equal(dropped, np.int32(new) - n_out)
        held_now = d.get(pp, (B, bps), np.int32)
        assert np.array_equal((held_now >= 0).sum(1), -(-kept // bs))
        assert d.get(n, (1,), np.int32)[0] == 12 - int((-(-kept // bs)).sum() - (-(-past // bs)).sum())
