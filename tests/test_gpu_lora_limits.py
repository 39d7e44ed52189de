"""Adapters by request (slhip_lora) at the limits of its numbers and sizes."""
import numpy as np
import pytest

from sharplight_amd import native
from tests import step_ref
from tests.devutil import Dev, log
from tests.test_gpu_lora import NP, TYPES, Case, held, values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("x,w,y", TYPES)
@pytest.mark.parametrize("new,rank", [(1, 16), (3, 40), (70, 16), (70, 33)])
def test_h_keeps_its_24_bits(device, new, rank, x, w, y):
    """h = (1 + 2^-10 + 2^-20, -1, -2^-10) whose sum is 2^-20: what is held of h in 16 bits leaves 0 of it."""
    K, N = 64, 72
    c = Case("bits", [new], [0], 1, rank, K, N, x, w, y)
    c.vx[:], c.va[:], c.vb[:], c.vadd[:] = 0, 0, 0, 0
    c.vx[:, :3] = [1.0, 2.0 ** -10, 2.0 ** -20]
    c.va[0, 0, :3], c.va[0, 1, 0], c.va[0, rank - 1, 1] = 1.0, -1.0, -1.0
    c.vb[0, :, [0, 1, rank - 1]] = 1.0
    (c.x, c.vx), (c.a, c.va), (c.b, c.vb), (c.add, c.vadd) = (held(v, t) for v, t in ((c.vx, x), (c.va, w), (c.vb, w), (c.vadd, y)))
    with Dev() as d:
        args, more = c.put(d)
        log(f"lora bits of h {x}/{w}/{y} rank={rank} rows={new}")
        native.lora(*args, **more)
        native.synchronize()
        got = values(d.get(c.py, (c.T, N), NP[y]), y)
    assert (got == 2.0 ** -20).all(), got[0, :4]


@pytest.mark.parametrize("x,w,y", TYPES)
def test_rows_beside_ones_that_are_not_finite(device, x, w, y):
    """Within the bound of their own type's result."""
    c = Case("beside", [40, 1, 1], [0, 1, 1], 2, 16, 64, 48, x, w, y)
    clean, bound = c.expected()
    bad = {7: np.inf, 20: np.nan, 41: -np.inf}
    for r, v in bad.items():
        c.x[r, 3] = held(np.float64([v]), x)[0][0]
    with Dev() as d:
        args, more = c.put(d)
        log(f"lora beside rows that are not finite {x}/{w}/{y}")
        native.lora(*args, **more)
        native.synchronize()
        got = values(d.get(c.py, (c.T, c.N), NP[y]), y)
    others = [t for t in range(c.T) if t not in bad]
    assert (np.abs(got - clean)[others] <= step_ref.rounded_bound(clean, bound, y)[others]).all()
    assert not np.isfinite(got[list(bad)]).any()


def test_more_rows_than_a_launch_has_thread_blocks(device):
    """2^29 rows and some: more 32-row tiles than the 2^24 thread blocks of a launch, so that thread blocks take turns. Most rows are of a
    request without an adapter, in place, so are not touched; the first and the last ones are compared."""
    T, K, N, R, few, requests = (1 << 29) + 100, 8, 8, 16, 50, 3
    rng = np.random.default_rng(3)
    starts = np.int32([0, few, T - few, T])
    adapter = np.int32([0, -1, 1])
    a, va = held(rng.standard_normal((2, R, K)), "bf16")
    b, vb = held(rng.standard_normal((2, N, R)) / 4, "bf16")
    ends = [held(rng.standard_normal((few, K)), "bf16") for _ in range(2)]
    adds = [held(rng.standard_normal((few, N)), "bf16") for _ in range(2)]
    with Dev() as d:
        x, y = d.empty(T * K * 2, fill=None), d.empty(T * N * 2, fill=None)
        for at, parts in ((x, ends), (y, adds)):
            for first, (bits, _) in zip((0, T - few), parts):
                native.call("slhip_memcpy_h2d", at + first * 16, bits.ctypes.data, bits.nbytes, None)
        near = np.full((few, N), 0x1234, np.uint16)  # rows next to them
        for first in (few, T - 2 * few):
            native.call("slhip_memcpy_h2d", y + first * 16, near.ctypes.data, near.nbytes, None)
        size = native.lora_work_bytes(T, R)
        log(f"lora of {T} rows, {size >> 30} GiB of workspace")
        native.lora("bf16", "bf16", x, y, y, native.lora_set("bf16", d.put(a), d.put(b), 2, R, K, N), native.lora_rows(requests, T, d.put(starts), d.put(adapter)),
                    work=d.empty(size, fill=None), work_bytes=size)
        native.synchronize()
        for i, first in enumerate((0, T - few)):
            got = values(d.get(y + first * 16, (few, N), np.uint16), "bf16")
            want, bound = step_ref.lora(ends[i][1], adds[i][1], va, vb, [0, few], [i])
            assert np.all(np.abs(got - want) <= step_ref.rounded_bound(want, bound, "bf16"))
        for first in (few, T - 2 * few):
            assert (d.get(y + first * 16, (few, N), np.uint16) == 0x1234).all()
