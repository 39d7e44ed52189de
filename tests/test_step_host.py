"""Host-side checks of adapters, draft verification and the block tables' step back: the arguments' layout, what the calls refuse before
any device work, workspaces, and the 64-bit statements that the GPU tests compare with, against values worked out by hand."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from sharplight_amd import native
from tests import kv8_ref, step_ref
from tests.test_kv8_host import FAKE, _pages

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_layouts_match_c(tmp_path):
    structs = {"slhip_drafts": native.Drafts, "slhip_lora_set": native.LoraSet, "slhip_lora_rows": native.LoraRows}
    lines = "".join(f'printf("{s}.{f} %zu\\n", offsetof({s}, {f}));' for s, c in structs.items() for f, _ in c._fields_)
    lines += "".join(f'printf("{s} %zu\\n", sizeof({s}));' for s in structs)
    src = tmp_path / "l.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "sharplight_hip.h"\nint main(void) {' + lines + "return 0; }")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o",
                    str(tmp_path / "l")], check=True)
    lay = dict(x.split() for x in subprocess.run([str(tmp_path / "l")], check=True, capture_output=True, text=True).stdout.splitlines())
    for s, c in structs.items():
        assert int(lay[s]) == ctypes.sizeof(c)
        for f, _ in c._fields_:
            assert int(lay[f"{s}.{f}"]) == getattr(c, f).offset, (s, f)


# ---- refusals ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kw,error,match", [
    (dict(block_size=24), ValueError, "power of two"), (dict(requests=-1), ValueError, "negative"),
    (dict(requests=4097), NotImplementedError, "4096 requests"), (dict(page_slots=131073), NotImplementedError, "131072"),
    (dict(blocks_per_slot=1 << 27), NotImplementedError, "2\\^31"), (dict(n_free_out=None), ValueError, "n_free"),
    (dict(free_blocks=None), ValueError, "free list"), (dict(past=None), ValueError, "past"), (dict(count=None), ValueError, "count"),
    (dict(pages=None), ValueError, "pages"),
])
def test_trim_refusals(kw, error, match):
    with pytest.raises(error, match=match):
        native.kv_pages_trim(_pages(**{"starts": None, **kw}))


def _set(**kw):
    a = dict(dtype="bf16", a=FAKE, b=FAKE, adapters=2, max_rank=8, K=64, N=32)
    a.update(kw)
    return native.lora_set(**a)


def _rows(**kw):
    a = dict(requests=2, tokens=4, starts=FAKE, adapter=FAKE)
    a.update(kw)
    return native.lora_rows(**a)


@pytest.mark.parametrize("sets,rows,call,error,match", [
    (dict(dtype=7), {}, {}, NotImplementedError, "dtype"), ({}, {}, dict(dtype_x="f16"), NotImplementedError, "dtypes"),
    ({}, {}, dict(dtype_y="f16"), NotImplementedError, "dtypes"), (dict(max_rank=257), {}, {}, NotImplementedError, "256 ranks"),
    (dict(max_rank=0), {}, {}, ValueError, "bad size"), (dict(K=0), {}, {}, ValueError, "bad size"), (dict(N=0), {}, {}, ValueError, "bad size"),
    (dict(adapters=-1), {}, {}, ValueError, "bad size"), (dict(K=7), {}, {}, NotImplementedError, "less than 8"),
    (dict(N=7), {}, {}, NotImplementedError, "less than 8"), (dict(N=1 << 24, max_rank=64), {}, {}, NotImplementedError, "2\\^31 bytes"), (dict(K=1 << 25), {}, {}, NotImplementedError, "too many"),
    ({}, dict(requests=4097), {}, NotImplementedError, "4096 requests"), ({}, dict(requests=-1), {}, ValueError, "bad size"),
    ({}, dict(tokens=1 << 31), {}, NotImplementedError, "too many"), ({}, dict(starts=None), {}, ValueError, "starts"),
    ({}, dict(adapter=None), {}, ValueError, "adapter"), ({}, {}, dict(x=None), ValueError, "x, y"), ({}, {}, dict(y=None), ValueError, "x, y"),
    (dict(a=None), {}, {}, ValueError, "a and b"), ({}, {}, dict(x_stride=63), ValueError, "stride"), ({}, {}, dict(y_stride=31), ValueError, "stride"),
    ({}, {}, dict(add_stride=31), ValueError, "stride"), (dict(a_stride=511), {}, {}, ValueError, "adapter stride"),
    (dict(b_stride=255), {}, {}, ValueError, "adapter stride"), ({}, {}, dict(work=None), ValueError, "workspace"),
    ({}, {}, dict(work=FAKE + 4), ValueError, "workspace"), ({}, {}, dict(work_bytes=64), ValueError, "workspace"),
    ({}, {}, dict(add=FAKE, y=FAKE, y_stride=40), ValueError, "another stride"),
    ({}, {}, dict(y_stride=1 << 30), NotImplementedError, "2\\^30"), ({}, {}, dict(add_stride=1 << 30), NotImplementedError, "2\\^30"),
    ({}, dict(tokens=(1 << 31) - (1 << 17)), {}, NotImplementedError, "too many"),
])
def test_lora_refusals(sets, rows, call, error, match):
    a = dict(dtype_x="f32", dtype_y="f32", x=FAKE, add=FAKE, y=FAKE + 4096, work=FAKE, work_bytes=1 << 40)
    a.update(call)
    with pytest.raises(error, match=match):
        native.lora(a.pop("dtype_x"), a.pop("dtype_y"), a.pop("x"), a.pop("add"), a.pop("y"), _set(**sets), _rows(**rows), **a)


def test_lora_of_nothing_needs_nothing():
    native.lora("f32", "f32", None, None, None, _set(), _rows(requests=0, starts=None, adapter=None))
    native.lora("f32", "f32", None, None, None, _set(), _rows(tokens=0))
    with pytest.raises(ValueError, match="required"):
        native.call("slhip_lora", 0, 0, FAKE, 64, FAKE, 32, FAKE, 32, None, None, None, 0, None)


def _drafts(**kw):
    a = dict(requests=2, tokens=4, vocab=100, starts=FAKE, ids=FAKE, accept=FAKE, sample=FAKE, out=FAKE, out_stride=4, n_out=FAKE)
    a.update(kw)
    return native.drafts(**a)


@pytest.mark.parametrize("kw,call,error,match", [
    ({}, dict(dtype="f16"), NotImplementedError, "dtype"), (dict(requests=-1), {}, ValueError, "bad size"), (dict(vocab=0), {}, ValueError, "bad size"),
    (dict(tokens=-1), {}, ValueError, "bad size"), (dict(requests=65537), {}, NotImplementedError, "too many"),
    (dict(vocab=(1 << 24) + 1), {}, NotImplementedError, "too many"), (dict(tokens=1 << 23), {}, NotImplementedError, "too many"),
    (dict(requests=4096, vocab=1 << 24), {}, NotImplementedError, "too many"), (dict(out_stride=-1), {}, ValueError, "stride"),
    ({}, dict(target_stride=99), ValueError, "stride"), ({}, dict(draft_stride=99), ValueError, "stride"), (dict(starts=None), {}, ValueError, "starts"),
    (dict(n_out=None), {}, ValueError, "n_out"), (dict(out=None), {}, ValueError, "out"), ({}, dict(target=None), ValueError, "target"),
    (dict(ids=None), {}, ValueError, "ids"), (dict(accept=None), {}, ValueError, "accept"), (dict(sample=None), {}, ValueError, "sample"),
    ({}, dict(work=None), ValueError, "workspace"), ({}, dict(work=FAKE + 8), ValueError, "workspace"), ({}, dict(work_bytes=100), ValueError, "workspace"),
])
def test_draft_verify_refusals(kw, call, error, match):
    a = dict(dtype="f32", target=FAKE, draft=FAKE, work=FAKE, work_bytes=1 << 40)
    a.update(call)
    with pytest.raises(error, match=match):
        native.draft_verify(a.pop("dtype"), a.pop("target"), a.pop("draft"), _drafts(**kw), **a)


def test_draft_verify_of_no_requests_needs_nothing():
    native.draft_verify("f32", None, None, _drafts(requests=0, tokens=0, starts=None, ids=None, accept=None, sample=None, out=None, n_out=None))
    with pytest.raises(ValueError, match="null"):
        native.call("slhip_draft_verify", 0, FAKE, 100, None, 0, None, None, 0, None)


def test_workspaces_take_every_smaller_step():
    rng = np.random.default_rng(5)
    assert native.lora_work_bytes(-1, 8) == native.lora_work_bytes(8, 0) == native.lora_work_bytes(8, 257) == -1
    assert native.draft_verify_work_bytes(1, 1, 0) == native.draft_verify_work_bytes(65537, 1, 10) == -1
    for _ in range(300):
        t, r = int(np.exp2(rng.uniform(0, 18))), int(rng.integers(1, 257))
        most = native.lora_work_bytes(t, r)
        assert 0 < most <= 4 * 256 * max(65536, t) + 16 + 140 * (t + 4096)
        for _ in range(20):
            assert native.lora_work_bytes(int(rng.integers(0, t + 1)), int(rng.integers(1, r + 1))) <= most
        b, t, v = int(rng.integers(1, 600)), int(rng.integers(1, 3000)), int(np.exp2(rng.uniform(0, 18)))
        most = native.draft_verify_work_bytes(b, t, v)
        for _ in range(20):
            assert 0 <= native.draft_verify_work_bytes(int(rng.integers(0, b + 1)), int(rng.integers(0, t + 1)), int(rng.integers(1, v + 1))) <= most


# ---- the statements, by hand ---------------------------------------------------------------------------------------

def test_lora_statement():
    x = np.array([[1.0, 2.0], [3.0, -1.0], [0.5, 0.5], [9.0, 9.0]])
    a = np.array([[[1.0, 1.0], [0.0, 2.0]], [[-1.0, 0.0], [5.0, 5.0]]])
    b = np.array([[[1.0, 0.0], [0.0, 1.0], [1.0, 1.0]], [[2.0, 7.0], [3.0, 7.0], [0.0, 7.0]]])
    add = np.ones((4, 3))
    y, bound = step_ref.lora(x, add, a, b, [0, 1, 2, 3], [0, 1, -1], rank=[2, 1], scale=[0.5, 2.0])
    # row 0: h = (3, 4), B h = (3, 4, 7); row 1: h = (-3), B h = (-6, -9, 0); row 2 has no adapter; row 3 no request
    assert np.array_equal(y[:3], [[2.5, 3.0, 4.5], [-11.0, -17.0, 1.0], [1.0, 1.0, 1.0]]) and np.isnan(y[3]).all()
    assert (bound[2] == 0).all() and (bound[:2] > 0).all() and (bound[:2] < 1e-4).all()


def test_verify_statement():
    ln = np.log
    target = np.array([ln([0.5, 0.25, 0.25]), ln([0.1, 0.1, 0.8]), ln([0.2, 0.3, 0.5])])
    draft = np.array([ln([0.8, 0.1, 0.1]), ln([0.1, 0.8, 0.1]), ln([1 / 3] * 3)])
    go = lambda ids, accept, sample, d=draft, **kw: step_ref.verify(target, d, [0, 3], ids, accept, [sample], 3, **kw)  # noqa: E731
    # 0 accepted: 0.6 * 0.8 < 0.5; 1 refused: 0.2 * 0.8 > 0.1; what is left of row 1: (0, 0, 0.7)
    out, n, kept, dropped, lp, margin = go([9, 0, 1], [0.6, 0.2, 0.0], 0.9, past=[10])
    assert out.tolist() == [[0, 2, -1]] and n[0] == 2 and kept[0] == 12 and dropped[0] == 1
    assert np.allclose(lp, [[ln(0.5), ln(0.8), 0]]) and 0.01 < margin < 0.1
    # both accepted: the last row, 0.2 <= 0.45 < 0.5
    out, n, *_ = go([9, 0, 1], [0.6, 0.1, 0.0], 0.45)
    assert out.tolist() == [[0, 1, 1]] and n[0] == 3
    # chosen drafts: accepted below p alone; the refused one leaves the others
    out, n, *_ = go([9, 0, 1], [0.49, 0.11, 0.0], 0.1, d=None)
    assert out.tolist() == [[0, 0, -1]]
    # greedy
    out, n, *_ = go([9, 0, 1], [0.99, 0.99, 0.0], 0.1, tau=[0.0])
    assert out.tolist() == [[0, 2, -1]]
    out, n, _, _, lp, _ = step_ref.verify(np.array([[0.0, np.nan]]), None, [0, 1], [0], [0.5], [0.5], 2)
    assert out.tolist() == [[-1, -1]] and n[0] == 1 and np.isnan(lp[0, 0])


def test_trim_statement():
    pages = np.int32([[5, 6, 7, -1], [1, 2, -1, -1]])
    free = np.int32([9, 8, 0, 0, 0])
    # request 0 keeps 17 of 40 tokens (2 of 3 blocks), request 1 none of 32
    ok, p, f, n = step_ref.trim([17, 0], [23, 32], [0, 1], pages, 16, free, 2)
    assert ok and n == 5 and p.tolist() == [[5, 6, -1, -1], [-1, -1, -1, -1]] and f.tolist() == [9, 8, 2, 1, 7]
    assert not step_ref.trim([17, 0], [47, 32], [0, 1], pages, 16, free, 2)[0]  # an entry that is not there
    assert not step_ref.trim([17, 0], [23, 32], [0, 1], pages, 16, free, 3)[0]  # no room
    # an advance that is taken back leaves the list as it was
    ok, p, n, *_ = kv8_ref.advance([17, 5], [40, 30], [0, 1], np.int32([[5, 6, -1, -1], [1, -1, -1, -1]]), 16, np.int32([3, 4, 7, 8, 9]), 5, 70)
    assert ok and n == 1
    ok, p, f, n = step_ref.trim([17, 5], [40, 30], [0, 1], p, 16, np.int32([3, 0, 0, 0, 0]), n)
    assert ok and n == 5 and f.tolist() == [3, 4, 7, 8, 9] and p.tolist() == [[5, 6, -1, -1], [1, -1, -1, -1]]
