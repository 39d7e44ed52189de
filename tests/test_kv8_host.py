"""Host-side checks of the paged 8-bit cache: the work-item map, the arguments' layout, what the calls refuse before any
device work, and the 64-bit statements that the GPU tests compare with, against values worked out by hand."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from sharplight_amd import native
from tests import kv8_ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAKE = 0x1000  # never dereferenced: every call below fails validation first


def test_item_map(tmp_path):
    exe = tmp_path / "kv8_map_check"
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-fsanitize=address,undefined", "-o", str(exe),
                    os.path.join(ROOT, "tests", "kv8_map_check.cpp")], check=True, capture_output=True, timeout=300)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.split() == ["cases", "4000"]


def test_struct_layouts_match_c(tmp_path):
    structs = {"slhip_kv_pages": native.KvPages, "slhip_kv8_cache": native.Kv8Cache, "slhip_kv8_batch": native.Kv8Batch,
               "slhip_kv8_attn": native.Kv8Attn}
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


def _pages(**kw):
    a = dict(requests=2, past=FAKE, count=FAKE, pages=FAKE, page_slots=4, blocks_per_slot=8, block_size=16, free_blocks=FAKE,
             free_capacity=32, n_free=FAKE, n_free_out=FAKE, tokens=8, starts=FAKE)
    a.update(kw)
    return native.kv_pages(**a)


@pytest.mark.parametrize("kw,error,match", [
    (dict(block_size=24), ValueError, "power of two"), (dict(block_size=0), ValueError, "power of two"),
    (dict(requests=-1), ValueError, "negative"), (dict(requests=4097), NotImplementedError, "4096 requests"),
    (dict(page_slots=131073), NotImplementedError, "131072"), (dict(blocks_per_slot=1 << 27), NotImplementedError, "2\\^31"),
    (dict(n_free=None), ValueError, "n_free"), (dict(n_free_out=None), ValueError, "n_free"),
    (dict(free_blocks=None), ValueError, "free list"), (dict(past=None), ValueError, "past"), (dict(pages=None), ValueError, "pages"),
    (dict(tokens=1 << 31), NotImplementedError, "2\\^31"),
])
def test_kv_pages_refusals(kw, error, match):
    for call in (native.kv_pages_advance, native.kv_pages_release):
        with pytest.raises(error, match=match):
            call(_pages(**kw))


def test_kv_pages_advance_refusals():
    with pytest.raises(ValueError, match="count"):
        native.kv_pages_advance(_pages(count=None))
    with pytest.raises(ValueError, match="starts"):
        native.kv_pages_advance(_pages(starts=None))
    with pytest.raises(ValueError, match="null"):
        native.call("slhip_kv_pages_advance", None, None)


def _cache(**kw):
    a = dict(fmt="i8", k=FAKE, v=FAKE, k_scale=FAKE, v_scale=FAKE, blocks=8, block_size=16, heads=2, head_dim=64)
    a.update(kw)
    return native.kv8_cache(**a)


def _batch(**kw):
    a = dict(requests=2, tokens=4, starts=FAKE, past=FAKE, pages=FAKE, page_slots=2, blocks_per_slot=4)
    a.update(kw)
    return native.kv8_batch(**a)


CACHE_REFUSALS = [
    (dict(fmt=7), {}, NotImplementedError, "format"), (dict(head_dim=72), {}, NotImplementedError, "multiple of 16"),
    (dict(head_dim=272), {}, NotImplementedError, "up to 256"), (dict(head_dim=0), {}, ValueError, "bad size"),
    (dict(block_size=8), {}, NotImplementedError, "block size"), (dict(block_size=48), {}, NotImplementedError, "block size"),
    (dict(block_size=512), {}, NotImplementedError, "block size"), (dict(heads=0), {}, ValueError, "bad size"),
    (dict(blocks=0), {}, ValueError, "no blocks"), (dict(k=FAKE + 8), {}, ValueError, "aligned"),
    (dict(v=None), {}, ValueError, "codes and scales"), (dict(k_scale=None), {}, ValueError, "codes and scales"),
    ({}, dict(starts=None), ValueError, "starts"), ({}, dict(pages=None), ValueError, "pages"),
    ({}, dict(past=None), ValueError, "past"), ({}, dict(requests=-1), ValueError, "bad size"),
    ({}, dict(tokens=-1), ValueError, "bad size"), ({}, dict(tokens=1 << 31), NotImplementedError, "too many"),
    ({}, dict(blocks_per_slot=1 << 27), NotImplementedError, "too many"), ({}, dict(requests=65537), NotImplementedError, "too many"),
]


@pytest.mark.parametrize("cache,batch,error,match", CACHE_REFUSALS)
def test_cache_and_batch_refusals(cache, batch, error, match):
    with pytest.raises(error, match=match):
        native.kv8_write("bf16", FAKE, FAKE, _cache(**cache), _batch(**batch))
    with pytest.raises(error, match=match):
        native.kv8_attention("bf16", FAKE, FAKE, 4, _cache(**cache), _batch(**batch), scale=1.0, work=FAKE, work_bytes=1 << 40)


def test_write_refusals():
    with pytest.raises(NotImplementedError, match="dtype"):
        native.kv8_write("f16", FAKE, FAKE, _cache(), _batch())
    with pytest.raises(ValueError, match="k and v"):
        native.kv8_write("f32", None, FAKE, _cache(), _batch())
    with pytest.raises(ValueError, match="stride"):
        native.kv8_write("f32", FAKE, FAKE, _cache(), _batch(), v_stride_h=32)
    with pytest.raises(ValueError, match="stride"):
        native.kv8_write("f32", FAKE, FAKE, _cache(), _batch(), k_stride_t=-1)
    with pytest.raises(ValueError, match="required"):
        native.call("slhip_kv8_write", 0, FAKE, 128, 64, FAKE, 128, 64, None, None, None)


def test_attention_refusals():
    go = lambda q_heads=4, dtype="f32", q=FAKE, y=FAKE, work=FAKE, work_bytes=1 << 40, cache=None, **kw: native.kv8_attention(  # noqa: E731
        dtype, q, y, q_heads, cache or _cache(), _batch(blocks_per_slot=1000), scale=kw.pop("scale", 1.0), work=work, work_bytes=work_bytes, **kw)
    with pytest.raises(ValueError, match="multiple of 2"):
        go(q_heads=3)
    with pytest.raises(NotImplementedError, match="64 query heads"):
        go(q_heads=130)
    with pytest.raises(NotImplementedError, match="dtype"):
        go(dtype="f16")
    with pytest.raises(ValueError, match="q and y"):
        go(q=None)
    with pytest.raises(ValueError, match="stride"):
        go(q_stride_h=8)
    for kw in (dict(softcap=-1.0), dict(softcap=float("nan")), dict(softcap=float("inf")), dict(scale=float("nan")),
               dict(scale=float("inf")), dict(window=-1), dict(max_new=-1)):
        with pytest.raises(ValueError, match="finite"):
            go(**kw)
    with pytest.raises(ValueError, match="workspace has 0 bytes"):
        go(work=None)
    with pytest.raises(ValueError, match="workspace has 64 bytes"):
        go(work_bytes=64)
    with pytest.raises(ValueError, match="workspace"):
        go(work=FAKE + 4)


def test_attention_refuses_more_keys_than_its_sums_hold():
    batch = lambda requests: _batch(requests=requests, page_slots=1 << 16, tokens=1 << 16, blocks_per_slot=(1 << 23) // 16)  # noqa: E731
    with pytest.raises(NotImplementedError, match="are too many"):
        native.kv8_attention("f32", FAKE, FAKE, 4, _cache(), batch(1 << 16), scale=1.0, max_new=1, work=FAKE, work_bytes=1 << 40)
    assert native.kv8_attention_work_bytes(4, _cache(), batch(1 << 16), 1) == -1
    assert native.kv8_attention_work_bytes(4, _cache(), batch(1 << 15), 1) > 0


def test_launches_past_their_limits_are_refused():
    """A launch has less than 2^32 threads."""
    most = _batch(tokens=(1 << 31) - (1 << 17), blocks_per_slot=1000)
    with pytest.raises(NotImplementedError, match="too many rows"):
        native.kv8_write("bf16", FAKE, FAKE, _cache(), most)
    go = lambda cache, batch, q_heads, **kw: native.kv8_attention("bf16", FAKE, FAKE, q_heads, cache, batch, scale=1.0, work=FAKE,  # noqa: E731
                                                                  work_bytes=1 << 40, **kw)
    with pytest.raises(NotImplementedError, match="too many tiles"):
        go(_cache(), most, 4)
    for slots in (4, 1000):  # short contexts, and such that are shared out
        with pytest.raises(NotImplementedError, match="too many tiles"):
            go(_cache(heads=4096), _batch(requests=65536, page_slots=65536, tokens=65536, blocks_per_slot=slots), 4096, max_new=1)


def test_work_bytes():
    need = native.kv8_attention_work_bytes(4, _cache(), _batch(blocks_per_slot=1000), 1)
    assert 0 < need < 1 << 28
    assert native.kv8_attention_work_bytes(4, _cache(), _batch(), 1) == 0  # contexts of 64 tokens at most: one launch
    assert native.kv8_attention_work_bytes(4, _cache(), _batch(requests=0), 1) == 0
    assert native.kv8_attention_work_bytes(3, _cache(), _batch(), 1) == -1
    for tokens in (1, 31, 512, 100000):
        for d in (64, 80, 128, 256):
            for max_new in (0, 1, 5, tokens):
                assert 0 <= native.kv8_attention_work_bytes(8, _cache(head_dim=d), _batch(tokens=tokens, blocks_per_slot=10000), max_new) < 1 << 28


def test_empty_calls_need_nothing():
    native.kv8_write("f32", None, None, _cache(k=None), _batch(tokens=0, starts=None))
    native.kv8_attention("f32", None, None, 4, _cache(k=None), _batch(requests=0, starts=None), scale=1.0)


# ---- the 64-bit statements -----------------------------------------------------------------------------------------

def test_codes_by_hand():
    t = kv8_ref.code_values("e4m3")
    assert (t[0], t[1], t[8], t[0x38], t[0x7E], t[0xFE]) == (0.0, 2.0 ** -9, 2.0 ** -6, 1.0, 448.0, -448.0) and np.isnan(t[0x7F])
    # ties go to even codes: 1.0625 between 1 (0x38) and 1.125 (0x39); 1.1875 between 0x39 and 0x3A; half the smallest to 0
    assert list(kv8_ref.to_codes(np.array([1.0625, 1.1875, 2.0 ** -10, 1.5 * 2.0 ** -9, -1.0, -2.0 ** -11, 447.9]), "e4m3")) == [
        0x38, 0x3A, 0, 2, 0xB8, 0x80, 0x7E]
    assert list(kv8_ref.to_codes(np.array([0.5, 1.5, -2.5, 126.6]), "i8").view(np.int8)) == [0, 2, -2, 127]
    assert kv8_ref.scale_of(127.0, "i8") == 1 and kv8_ref.scale_of(127.5, "i8") == 2 and kv8_ref.scale_of(448.0, "e4m3") == 1
    assert kv8_ref.scale_of(0.0, "i8") == 2.0 ** -40 and np.isnan(kv8_ref.scale_of(127.01 * 2.0 ** 40, "i8"))


def test_write_by_hand():
    c = kv8_ref.Cache("i8", 3, 16, 1, 16)
    pages = np.array([[2, 0]])
    k = np.zeros((2, 1, 16))
    k[0, 0, 0], k[1, 0, 0] = 3.0, 100.0
    kv8_ref.write(c, k, k, [0, 1], [15], [0], pages)  # the last token of a block that was begun before
    assert c.ks[2, 0] == 2.0 ** -5 and c.k[2, 0, 15, 0] == 96 and c.v[2, 0, 0, 0, 15] == 96
    kv8_ref.write(c, k, k, [0, 2], [15], [0], pages)  # again, and the next block's first
    assert c.ks[2, 0] == 2.0 ** -5 and c.ks[0, 0] == 1.0 and c.k[0, 0, 0, 0] == 100
    k[0, 0, 0] = 200.0
    kv8_ref.write(c, k, k, [0, 1], [1], [0], pages)  # grows by 2^6: 96 steps of before are 1.5 now, and go to 2
    assert c.ks[2, 0] == 2.0 and c.k[2, 0, 1, 0] == 100 and c.k[2, 0, 15, 0] == 2


def test_attention_by_hand():
    """One key: y is its value; two equal keys: their mean; a window of one: the own value."""
    c = kv8_ref.Cache("i8", 1, 16, 1, 16)
    c.k[0, 0, :2], c.ks[:], c.vs[:] = 1, 1.0, 0.5
    c.v[0, 0, 0, :, 0], c.v[0, 0, 0, :, 1] = 10, 30
    q = np.ones((2, 1, 16))
    y, b = kv8_ref.attention(c, q, [0, 2], [0], [0], np.array([[0]]), scale=1.0)
    assert np.allclose(y[0], 5.0) and np.allclose(y[1], 10.0) and (b > 0).all() and (b < 1e-3).all()
    y, _ = kv8_ref.attention(c, q, [0, 2], [0], [0], np.array([[0]]), scale=1.0, window=1)
    assert np.allclose(y[1], 15.0)
    y, _ = kv8_ref.attention(c, q, [0, 2], [0], [0], np.array([[-1]]), scale=1.0)
    assert (y == 0).all()


def test_tables_by_hand():
    pages = np.full((3, 2), -1)
    ok, p, n, starts, seq, pos = kv8_ref.advance([0, 16], [17, 1], [2, 0], pages, 16, np.arange(10, 16), 5, 20)
    assert ok and n == 2 and list(p[2]) == [14, 13] and list(p[0]) == [-1, 12] and list(starts) == [0, 17, 18]
    assert list(seq[16]) == [2, 16, 0, 13] and list(seq[17]) == [0, 16, 1, 12] and list(seq[18]) == [-1] * 4 and pos[17] == 16
    ok, p, f, n = kv8_ref.release([17], [2], p, 16, np.arange(10, 16), 2)
    assert ok and n == 4 and list(f) == [10, 11, 14, 13, 14, 15] and list(p[2]) == [-1, -1]
