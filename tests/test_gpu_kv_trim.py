"""GPU parity of the block tables' step back (slhip_kv_pages_trim): whole numbers, equal to tests/step_ref.py."""
import numpy as np
import pytest

from sharplight_amd import native
from tests import kv8_ref, step_ref
from tests.devutil import Dev, log
from tests.test_gpu_lora import rng_of

pytestmark = pytest.mark.gpu


def _tables(rng, B, bs, most_past, most_back, slots):
    past, count = (rng.integers(0, m + 1, B).astype(np.int32) for m in (most_past, most_back))
    past[: B // 3] -= past[: B // 3] % bs
    bps = max(-(-(most_past + most_back) // bs), 1)
    slot = rng.permutation(slots)[:B].astype(np.int32)
    pages = np.full((slots, bps), -1, np.int32)
    ids = iter(rng.permutation(B * bps + 100).astype(np.int32))
    for i in range(B):
        for j in range(-(-(int(past[i]) + int(count[i])) // bs)):
            pages[slot[i], j] = next(ids)
    back = sum(-(-(int(p) + int(c)) // bs) - -(-int(p) // bs) for p, c in zip(past, count))
    free = np.full(back + 9, -7, np.int32)
    free[:5] = [next(ids) for _ in range(5)]
    return past, count, slot, pages, free, back


def _trim(d, past, count, slot, pages, bs, free, n_free, in_place=False, with_slots=True):
    at = {"pages": d.put(pages), "free": d.put(free), "n": d.put(np.int32([n_free])), "out": d.put(np.int32([77]))}
    if in_place:
        at["out"] = at["n"]
    p = native.kv_pages(len(past), d.put(past), d.put(count), at["pages"], pages.shape[0], pages.shape[1], bs, at["free"], len(free), at["n"], at["out"],
                        slots=d.put(slot) if with_slots else None)
    return p, at


def _check(d, at, want):
    ok, pages, free, n = want
    assert np.array_equal(d.get(at["pages"], pages.shape, np.int32), pages)
    assert np.array_equal(d.get(at["free"], free.shape, np.int32), free)
    assert d.get(at["out"], (1,), np.int32)[0] == n
    return ok


@pytest.mark.parametrize("B,bs,most_past,most_back,in_place", [
    (1, 16, 0, 1, True), (1, 16, 40, 40, False), (3, 1, 5, 3, True), (64, 16, 500, 4, True), (65, 32, 300, 40, False), (333, 64, 1000, 300, True),
    (1100, 16, 50, 20, False), (4096, 16, 33, 5, True), (7, 16, 100, 1500, True), (40, 128, 900, 4000, False), (5, 16, 20, 0, True),
    (9, 16, 100, 50000, True)])
def test_trim(device, B, bs, most_past, most_back, in_place):
    rng = rng_of("trim", B, bs, most_past, most_back)
    past, count, slot, pages, free, back = _tables(rng, B, bs, most_past, most_back, B + 3)
    with Dev() as d:
        log(f"kv_pages_trim B={B} bs={bs} back={back}")
        p, at = _trim(d, past, count, slot, pages, bs, free, 5, in_place)
        native.kv_pages_trim(p)
        native.synchronize()
        assert _check(d, at, step_ref.trim(past, count, slot, pages, bs, free, 5))


def test_no_requests_and_no_slots(device):
    rng = rng_of("none")
    with Dev() as d:
        log("kv_pages_trim of nothing")
        p, at = _trim(d, np.int32([]), np.int32([]), np.int32([]), np.full((2, 2), 5, np.int32), 16, np.int32([1, 2]), 1)
        native.kv_pages_trim(p)
        native.synchronize()
        assert d.get(at["out"], (1,), np.int32)[0] == 1
        past, count, _, pages, free, _ = _tables(rng, 6, 16, 60, 60, 6)
        order = np.arange(6, dtype=np.int32)
        for i in range(6):
            n = -(-(int(past[i]) + int(count[i])) // 16)
            pages[i] = -1
            pages[i, :n] = 100 * i + np.arange(n)
        log("kv_pages_trim without slots")
        p, at = _trim(d, past, count, order, pages, 16, free, 5, with_slots=False)
        native.kv_pages_trim(p)
        native.synchronize()
        assert _check(d, at, step_ref.trim(past, count, order, pages, 16, free, 5))


@pytest.mark.parametrize("bad", ["length", "count", "outgrown", "slot", "twice", "room", "entry", "count of free"])
@pytest.mark.parametrize("B", [5, 70])
def test_all_or_nothing(device, bad, B):
    rng = rng_of("bad", bad, B)
    past, count, slot, pages, free, back = _tables(rng, B, 16, 100, 60, B + 3)
    count[B - 2] = 40
    pages[slot[B - 2], : -(-(int(past[B - 2]) + 40) // 16)] = 9
    back = sum(-(-(int(p) + int(c)) // 16) - -(-int(p) // 16) for p, c in zip(past, count))
    n_free, free = 5, np.full(5 + back, 3, np.int32)
    if bad == "length":
        past[2] = -1
    elif bad == "count":
        count[2] = -1
    elif bad == "outgrown":
        count[2] = pages.shape[1] * 16 + 1
    elif bad == "slot":
        slot[2] = B + 3
    elif bad == "twice":
        slot[2] = slot[0]
    elif bad == "room":
        free = free[:-1]
    elif bad == "entry":
        pages[slot[B - 2], (int(past[B - 2]) + 39) // 16] = -1
    else:
        n_free = len(free) + 1
    with Dev() as d:
        log(f"kv_pages_trim bad {bad} B={B}")
        p, at = _trim(d, past, count, slot, pages, 16, free, n_free)
        native.kv_pages_trim(p)
        with pytest.raises(native.SlhipCacheError):
            native.synchronize()
        native.synchronize()
        want = step_ref.trim(past, count, slot, pages, 16, free, n_free)
        assert not want[0]
        _check(d, at, want)


@pytest.mark.parametrize("B", [3, 100, 700])
def test_an_advance_taken_back(device, B):
    """What an advance took goes back whole: tables, list and count are as before; then in parts, and the blocks are taken again."""
    rng = rng_of("back", B)
    bs, bps = 16, 40
    past, count = rng.integers(0, 400, B).astype(np.int32), rng.integers(0, 200, B).astype(np.int32)
    pages = np.full((B, bps), -1, np.int32)
    ids = iter(rng.permutation(B * bps + 50).astype(np.int32))
    for i in range(B):
        for j in range(-(-int(past[i]) // bs)):
            pages[i, j] = next(ids)
    free = np.int32([next(ids) for _ in range(B * 14 + 7)])
    with Dev() as d:
        n = d.put(np.int32([len(free)]))
        pp, pf, pc = d.put(pages), d.put(free), d.put(count)
        T = int(count.sum())
        starts = d.empty(4 * (B + 1))
        a = native.kv_pages(B, d.put(past), pc, pp, B, bps, bs, pf, len(free), n, n, T, starts)
        log(f"advance and trim B={B}")
        native.kv_pages_advance(a)
        native.kv_pages_trim(a)
        native.synchronize()
        assert np.array_equal(d.get(pp, pages.shape, np.int32), pages) and np.array_equal(d.get(pf, free.shape, np.int32), free)
        assert d.get(n, (1,), np.int32)[0] == len(free)
        kept = (past + rng.integers(0, count + 1)).astype(np.int32)
        t = native.kv_pages(B, d.put(kept), d.put((past + count - kept).astype(np.int32)), pp, B, bps, bs, pf, len(free), n, n)
        native.kv_pages_advance(a)
        native.kv_pages_trim(t)
        native.synchronize()
        ok, p1, n1, *_ = kv8_ref.advance(past, count, np.arange(B), pages, bs, free, len(free), T)
        ok2, p2, f2, n2 = step_ref.trim(kept, past + count - kept, np.arange(B), p1, bs, free, n1)
        assert ok and ok2
        assert np.array_equal(d.get(pp, pages.shape, np.int32), p2) and np.array_equal(d.get(pf, free.shape, np.int32), f2)
        assert d.get(n, (1,), np.int32)[0] == n2
        held = p2[p2 >= 0]
        assert len(set(held)) == len(held) and not set(held) & set(f2[:n2])


@pytest.mark.parametrize("total", [1, 1023, 1024, 1025, 4096, 4097, 16384, 16385])
@pytest.mark.parametrize("B", [5, 900, 4096])
def test_numbers_of_blocks(device, B, total):
    """Trims and releases of exactly so many blocks, spread over few and many requests, empty ones among them."""
    rng = rng_of("numbers", B, total)
    back = np.bincount(rng.choice(np.append(rng.permutation(B)[: B // 2], B - 1), total), minlength=B)
    keep = rng.integers(0, 3, B)
    bs, bps = 16, int((back + keep).max()) + 1
    past = (keep * bs).astype(np.int32)
    count = (back * bs - np.where(back > 0, rng.integers(0, bs, B), 0)).astype(np.int32)
    slot = rng.permutation(B + 5)[:B].astype(np.int32)
    pages = np.full((B + 5, bps), -1, np.int32)
    ids = iter(rng.permutation(int((back + keep).sum()) + 3).astype(np.int32))
    for i in range(B):
        for j in range(int(back[i] + keep[i])):
            pages[slot[i], j] = next(ids)
    with Dev() as d:
        free = np.full(total + 4, -7, np.int32)
        free[:2] = [next(ids) for _ in range(2)]
        log(f"kv_pages_trim of {total} blocks, B={B}")
        p, at = _trim(d, past, count, slot, pages, bs, free, 2)
        native.kv_pages_trim(p)
        native.synchronize()
        assert _check(d, at, step_ref.trim(past, count, slot, pages, bs, free, 2))
        past = (back * bs - np.where(back > 0, rng.integers(0, bs, B), 0)).astype(np.int32)
        log(f"kv_pages_release of {total} blocks, B={B}")
        p, at = _trim(d, past, count, slot, pages, bs, free, 2)
        native.kv_pages_release(p)
        native.synchronize()
        assert _check(d, at, kv8_ref.release(past, slot, pages, bs, free, 2))
