"""A serving step of requests with adapters, a paged 8-bit cache and drafted tokens, as a program would record it once and replay it: block
tables forward, embeddings, projections with each request's adapter, rotation, cache write and attention, logits, the drafts' verification, block
tables back. After every replay each operator's result is compared with its 64-bit statement on the inputs that it had on the device."""
import numpy as np
import pytest

from sharplight_amd import native
from tests import kv8_ref, step_ref
from tests.devutil import Dev, log
from tests.test_gpu_draft import NEAR
from tests.test_gpu_lora import held, rng_of, values

pytestmark = pytest.mark.gpu

B, SLOTS, T, BS, BPS, BLOCKS = 5, 7, 18, 16, 6, 24
E, HEADS, KV_HEADS, D, V, ADAPTERS, R, STRIDE = 192, 4, 2, 64, 1003, 3, 16, 6


class Model:
    """Weights, buffers and the step's calls."""

    def __init__(self, d, rng, fmt):
        self.d = d
        bf16 = lambda *s, size=1.0: held(rng.standard_normal(s) * (size / np.sqrt(s[-1])), "bf16")  # noqa: E731
        self.table = d.put(bf16(V, E, size=E ** 0.5)[0])
        width = {"q": HEADS * D, "k": KV_HEADS * D, "v": KV_HEADS * D}
        self.w = {k: d.put(bf16(n, E)[0]) for k, n in width.items()} | {"o": d.put(bf16(E, HEADS * D)[0]), "head": d.put(bf16(V, E, size=3.0)[0])}
        self.ranks, self.scale = np.int32([R, 7, 12]), np.float32([0.5, 2.0, 1.0])
        pr, ps = d.put(self.ranks), d.put(self.scale)
        self.lora, self.lora_values = {}, {}
        for k, (n_in, n_out) in {"q": (E, HEADS * D), "o": (HEADS * D, E)}.items():
            a, va = bf16(ADAPTERS, R, n_in)
            b, vb = bf16(ADAPTERS, n_out, R)
            self.lora[k] = native.lora_set("bf16", d.put(a), d.put(b), ADAPTERS, R, n_in, n_out, rank=pr, scale=ps)
            self.lora_values[k] = va, vb
        self.width = dict(width, x=E, base=HEADS * D, lora_q=HEADS * D, a=HEADS * D, o=E)
        self.at = {k: d.empty(2 * T * n) for k, n in self.width.items()}
        self.at |= {k: d.empty(4 * n) for k, n in (("z", T * V), ("starts", B + 1), ("pos", T), ("seq", 4 * T), ("ids", T), ("adapter", B), ("past", B),
                                                  ("count", B), ("slots", B), ("pages", SLOTS * BPS), ("free", BLOCKS), ("n_free", 1), ("accept", T),
                                                  ("sample", B), ("tau", B), ("q_logits", T * V), ("out", B * STRIDE), ("n_out", B), ("kept", B),
                                                  ("dropped", B), ("logp", B * STRIDE))}
        self.cache = kv8_ref.Cache(fmt, BLOCKS, BS, KV_HEADS, D, fill=rng)
        self.codes = [d.put(x) for x in (self.cache.k, self.cache.v, self.cache.ks, self.cache.vs)]
        self.kv = native.kv8_cache(fmt, *self.codes, BLOCKS, BS, KV_HEADS, D)
        p = self.at
        tables = lambda past, count: native.kv_pages(B, past, count, p["pages"], SLOTS, BPS, BS, p["free"], BLOCKS, p["n_free"], p["n_free"], T, p["starts"],  # noqa: E731
                                                     seq=p["seq"], pos=p["pos"], slots=p["slots"])
        self.forward, self.back = tables(p["past"], p["count"]), tables(p["kept"], p["dropped"])
        self.batch = native.kv8_batch(B, T, p["starts"], p["past"], p["pages"], SLOTS, BPS, slots=p["slots"])
        self.rows = native.lora_rows(B, T, p["starts"], p["adapter"])
        self.drafts = native.drafts(B, T, V, p["starts"], p["ids"], p["accept"], p["sample"], p["out"], STRIDE, p["n_out"], temperature=p["tau"],
                                    past=p["past"], kept=p["kept"], dropped=p["dropped"], logp=p["logp"])
        # one workspace: the calls follow each other
        self.size = max(native.kv8_attention_work_bytes(HEADS, self.kv, self.batch), native.lora_work_bytes(T, R), native.draft_verify_work_bytes(B, T, V))
        self.work = d.empty(self.size)

    def step(self, stream):
        p, more = self.at, dict(work=self.work, work_bytes=self.size, stream=stream)
        native.kv_pages_advance(self.forward, stream=stream)
        native.gather("bf16", self.table, V, E, p["ids"], T, "bf16", p["x"], stream=stream)
        for k, to in (("q", "base"), ("k", "k"), ("v", "v")):
            native.matvec("bf16", "bf16", "bf16", p["x"], T, E, self.w[k], self.width[k], p[to], stream=stream)
        native.lora("bf16", "bf16", p["x"], p["base"], p["lora_q"], self.lora["q"], self.rows, **more)
        native.rope("bf16", "bf16", [dict(x=p["k"], y=p["k"], heads=KV_HEADS), dict(x=p["lora_q"], y=p["q"], heads=HEADS)], p["pos"], T, D, stream=stream)
        native.kv8_write("bf16", p["k"], p["v"], self.kv, self.batch, stream=stream)
        native.kv8_attention("bf16", p["q"], p["a"], HEADS, self.kv, self.batch, scale=D ** -0.5, **more)
        native.matvec("bf16", "bf16", "bf16", p["a"], T, HEADS * D, self.w["o"], E, p["o"], stream=stream)
        native.lora("bf16", "bf16", p["a"], p["o"], p["o"], self.lora["o"], self.rows, **more)
        native.matvec("bf16", "bf16", "f32", p["o"], T, E, self.w["head"], V, p["z"], stream=stream)
        native.draft_verify("f32", p["z"], p["q_logits"], self.drafts, **more)
        native.kv_pages_trim(self.back, stream=stream)

    def put(self, stream, state):
        """The step's inputs; the cache as it was before."""
        for k, v in state.items():
            native.call("slhip_memcpy_h2d", self.at[k], v.ctypes.data, v.nbytes, stream.handle)
        for at, v in zip(self.codes, (self.cache.k, self.cache.v, self.cache.ks, self.cache.vs)):
            native.call("slhip_memcpy_h2d", at, v.ctypes.data, v.nbytes, stream.handle)
        stream.sync()

    def get(self, k, shape, dtype=np.int32):
        return self.d.get(self.at[k], shape, dtype)

    def bits(self, k):
        return self.get(k, (T, self.width[k]), np.uint16)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_captured_step_of_requests_with_drafts(device, fmt):
    rng = rng_of("step", fmt)
    st = native.Stream()
    with Dev() as d:
        m = Model(d, rng, fmt)
        past, slots = np.int32([14, 0, 15, 30, 3]), rng.permutation(SLOTS)[:B].astype(np.int32)
        free, n_free = rng.permutation(BLOCKS).astype(np.int32), BLOCKS
        ok, pages, n_free, *_ = kv8_ref.advance(np.zeros(B, np.int32), past, slots, np.full((SLOTS, BPS), -1, np.int32), BS, free, n_free, int(past.sum()))
        q_logits = (rng.standard_normal((T, V)) * 1.5).astype(np.float32)
        graph, back = None, 0
        # requests that rest, that have no draft and that have up to five; what they keep varies
        for rep, count in enumerate([[6, 3, 1, 0, 5], [6, 1, 0, 4, 3], [1, 1, 1, 1, 1], [2, 6, 5, 3, 2], [6, 0, 0, 0, 6], [4, 4, 4, 3, 3],
                                     [0, 0, 6, 6, 6], [6, 6, 0, 6, 0], [0, 6, 6, 0, 6], [3, 4, 3, 4, 4]]):
            count = np.int32(count)
            used, starts = int(count.sum()), np.concatenate([[0], np.cumsum(count)]).astype(np.int32)
            state = dict(past=past, count=count, slots=slots, pages=pages, free=free, n_free=np.int32([n_free]), q_logits=q_logits,
                         adapter=rng.integers(-1, ADAPTERS, B).astype(np.int32), tau=np.float32([0, 0.7, 1, 0, 1.3]),
                         ids=rng.integers(0, V, T).astype(np.int32), accept=rng.random(T).astype(np.float32), sample=rng.random(B).astype(np.float32))
            # first runs for the logits: the first two drafts of some requests become the target's choices, and the random numbers are chosen so
            # that no choice is nearer than NEAR to another
            for first in range(3):
                log(f"step {fmt} {rep}: eager run {first} of {used} rows")
                m.put(st, state)
                m.step(st.handle)
                st.sync()
                z = m.get("z", (T, V), np.float32).astype(np.float64)
                for i in range(B):
                    if first < 2 and count[i] > first + 1 and i != 2:
                        state["ids"][starts[i] + first + 1] = z[starts[i] + first].argmax()
            for i in range(B):
                for _ in range(50):
                    one = step_ref.verify(z, q_logits.astype(np.float64), starts[i:i + 2], state["ids"], state["accept"].astype(np.float64),
                                          state["sample"][i:i + 1].astype(np.float64), STRIDE, state["tau"][i:i + 1])
                    if one[5] > NEAR:
                        break
                    state["accept"][starts[i]:starts[i + 1]], state["sample"][i] = rng.random(count[i]), rng.random()
                else:
                    raise AssertionError("no random numbers that settle the choices")
            m.put(st, state)
            if graph is None:
                log(f"step {fmt}: capture")
                graph = native.Graph(st, lambda: m.step(st.handle))
            log(f"step {fmt} {rep}: replay")
            graph.launch(st)
            st.sync()
            # block tables: forward, then back
            ok, middle, n_mid, starts_want, _, pos = kv8_ref.advance(past, count, slots, pages, BS, free, n_free, T)
            assert ok and np.array_equal(m.get("starts", (B + 1,)), starts_want) and np.array_equal(m.get("pos", (T,)), pos)
            z2 = m.get("z", (T, V), np.float32).astype(np.float64)
            assert np.array_equal(z2[:used], z[:used])
            out, n_out, kept, dropped, logp, _ = step_ref.verify(z2, q_logits.astype(np.float64), starts, state["ids"], state["accept"].astype(np.float64),
                                                                 state["sample"].astype(np.float64), STRIDE, state["tau"], past=past)
            assert np.array_equal(m.get("n_out", (B,)), n_out) and np.array_equal(m.get("kept", (B,)), kept) and np.array_equal(m.get("dropped", (B,)), dropped)
            got, lp = m.get("out", (B, STRIDE)), m.get("logp", (B, STRIDE), np.float32)
            for i in range(B):
                assert np.array_equal(got[i, :n_out[i]], out[i, :n_out[i]])
                for j in range(n_out[i]):
                    assert abs(lp[i, j] - logp[i, j]) <= step_ref.logp_bound(z2[starts[i] + j], float(state["tau"][i]), logp[i, j])
            ok, after, free_after, n_after = step_ref.trim(np.int32(kept), np.int32(dropped), slots, middle, BS, free, n_mid)
            back += n_after - n_mid
            assert ok and np.array_equal(m.get("pages", (SLOTS, BPS)), after) and np.array_equal(m.get("free", (BLOCKS,)), free_after)
            assert m.get("n_free", (1,))[0] == n_after
            assert sorted(set(after[after >= 0]) | set(free_after[:n_after])) == list(range(BLOCKS))  # none lost, none twice
            # adapters; the in-place one's sum is made once more beside it
            x, a, q, base, lora_q = (values(m.bits(k), "bf16") for k in ("x", "a", "q", "base", "lora_q"))
            y, bound = step_ref.lora(x, base, *m.lora_values["q"], starts, state["adapter"], m.ranks, m.scale, bf16_parts=True)
            assert np.all(np.abs(lora_q - y)[:used] <= step_ref.rounded_bound(y, bound, "bf16")[:used])
            native.matvec("bf16", "bf16", "bf16", m.at["a"], T, HEADS * D, m.w["o"], E, m.at["x"])
            native.synchronize()
            y, bound = step_ref.lora(a, values(m.bits("x"), "bf16"), *m.lora_values["o"], starts, state["adapter"], m.ranks, m.scale, bf16_parts=True)
            assert np.all(np.abs(values(m.bits("o"), "bf16") - y)[:used] <= step_ref.rounded_bound(y, bound, "bf16")[:used])
            # the cache, bit for bit, and its attention
            k, v = (values(m.bits(n), "bf16").reshape(T, KV_HEADS, D) for n in "kv")
            kv8_ref.write(m.cache, k, v, starts, past, slots, middle)
            held_codes = [d.get(at, c.shape, c.dtype) for at, c in zip(m.codes, (m.cache.k, m.cache.v, m.cache.ks, m.cache.vs))]
            for got, want in zip(held_codes, (m.cache.k, m.cache.v, m.cache.ks, m.cache.vs)):
                assert np.array_equal(got, want)
            y, bound = kv8_ref.attention(m.cache, q.reshape(T, HEADS, D), starts, past, slots, middle, scale=D ** -0.5, dtype="bf16")
            assert np.all(np.abs(a.reshape(T, HEADS, D) - y)[:used] <= bound[:used])
            past, pages, free, n_free = np.int32(kept), after, free_after, n_after
        assert back > 0, "no block went back"
        del graph
