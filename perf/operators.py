"""Performance cases of the paged 8-bit KV cache: its block tables, its write and the attention that reads it.

One serving step calls them in this order: ``kv_pages_advance`` takes the blocks that the step's new tokens need from the
free list and lays out the step's rows, ``kv8_write`` quantises the tokens' K and V into those blocks, ``kv8_attention``
reads them back. ``run`` makes those calls where ``own`` is true; otherwise it computes the same from elementary torch
operations. ``exact`` restates each operator in 64 bits, request by request.

The cache: codes of K as [blocks, heads, block_size, D] and of V as [blocks, heads, block_size/16, D, 16], int8 ("i8") or
OCP E4M3 ("e4m3"), with one power-of-two scale a block and head for each of the two; a value is code * scale.

Ranges that ``draw`` covers: 1 to 512 requests, from one token to long prompts, contexts to 131072 tokens, blocks of 16 to
128 tokens, 1 to 16 K/V heads with 1 to 8 query heads each, head dims 64 to 256, f32 and bf16 activations, both formats,
with and without a score cap, a window and distance slopes.
"""
import math

import torch

own = False

DEV = "cuda"
TORCH = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}
QMAX = {"i8": 127.0, "e4m3": 448.0}
LEAST = -40  # the smallest scale is 2^LEAST


def listed():
    return [
        # a decode step's tables: 64 sequences of up to 4096 tokens, one new token each
        {"name": "pages_decode", "op": "pages", "requests": 64, "new": 1, "new_least": 1, "past": 4096, "block": 16},
        # a step that mixes prompts of up to 200 tokens with running sequences, cut at odd lengths
        {"name": "pages_mixed", "op": "pages", "requests": 333, "new": 200, "new_least": 1, "past": 2048, "block": 32},
        # the K and V of a decode step (8 K/V heads of 128), appended to blocks that are partly full
        {"name": "write_decode", "op": "write", "requests": 64, "new": 1, "new_least": 1, "past": 512, "block": 16, "kv_heads": 8,
         "dim": 128, "dtype": "bf16", "format": "e4m3"},
        # the K and V of an 8192-token prompt
        {"name": "write_prefill", "op": "write", "requests": 1, "new": 8192, "new_least": 8192, "past": 0, "block": 16, "kv_heads": 8,
         "dim": 128, "dtype": "bf16", "format": "e4m3"},
        # chunks of several prompts from an f32 graph, ragged, int8 blocks of 64
        {"name": "write_chunks_f32", "op": "write", "requests": 23, "new": 180, "new_least": 3, "past": 300, "block": 64, "kv_heads": 4,
         "dim": 64, "dtype": "f32", "format": "i8"},
        # the smallest attention call: one chat's next token, where latency is most of it
        {"name": "attn_one", "op": "attention", "requests": 1, "new": 1, "new_least": 1, "past": 500, "block": 16, "kv_heads": 8,
         "group": 4, "dim": 128, "dtype": "bf16", "format": "e4m3", "cap": 0.0, "window": 0, "slopes": False},
        # a decode step over a batch of sequences of 1 to 4096 tokens
        {"name": "attn_decode", "op": "attention", "requests": 64, "new": 1, "new_least": 1, "past": 4095, "block": 16, "kv_heads": 8,
         "group": 4, "dim": 128, "dtype": "bf16", "format": "e4m3", "cap": 0.0, "window": 0, "slopes": False},
        # two long documents' next token in f32, int8 blocks of 64
        {"name": "attn_long_f32", "op": "attention", "requests": 2, "new": 1, "new_least": 1, "past": 131000, "block": 64, "kv_heads": 8,
         "group": 4, "dim": 128, "dtype": "f32", "format": "i8", "cap": 0.0, "window": 0, "slopes": False},
        # a few drafted tokens checked at once, capped scores and a sliding window
        {"name": "attn_drafts", "op": "attention", "requests": 16, "new": 6, "new_least": 3, "past": 9000, "block": 32, "kv_heads": 4,
         "group": 2, "dim": 256, "dtype": "bf16", "format": "i8", "cap": 50.0, "window": 4096, "slopes": False},
        # a long prompt's causal attention (32 query heads on 8 K/V heads)
        {"name": "attn_prefill", "op": "attention", "requests": 1, "new": 8192, "new_least": 8192, "past": 0, "block": 16, "kv_heads": 8,
         "group": 4, "dim": 128, "dtype": "bf16", "format": "e4m3", "cap": 0.0, "window": 0, "slopes": False},
        # ragged prompt chunks over what is cached already, f32, a head each, distance slopes
        {"name": "attn_chunks_f32", "op": "attention", "requests": 5, "new": 611, "new_least": 77, "past": 1500, "block": 16, "kv_heads": 12,
         "group": 1, "dim": 64, "dtype": "f32", "format": "i8", "cap": 0.0, "window": 0, "slopes": True},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["pages", "write", "write", "attention", "attention", "attention"])
    new = 1 if rng.random() < 0.4 else _log(rng, 2, 4096)
    c = {"op": op, "requests": _log(rng, 1, 512), "new": new, "new_least": _log(rng, 1, new), "past": _log(rng, 1, 131072) - 1,
         "block": rng.choice([16, 16, 32, 64, 128])}
    if op == "pages":
        while c["requests"] * (c["new"] + c["past"] // 16) > 1 << 20:
            c["requests"] = c["requests"] // 2 + (c["requests"] == 1)
            c["past"] //= 2
        return c
    c.update(kv_heads=rng.choice([1, 2, 4, 6, 8, 16]), dim=rng.choice([64, 64, 80, 96, 128, 128, 128, 192, 256]),
             dtype=rng.choice(["bf16", "bf16", "f32"]), format=rng.choice(["e4m3", "i8"]))
    if op == "write":  # no more values than the largest listed write has, and a cache that is quick to look at
        while c["requests"] * c["new"] * c["kv_heads"] * c["dim"] > 8192 * 1024:
            c["new"] = c["new"] // 2 + 1
            c["requests"] = c["requests"] // 2 + 1
        c["past"] = min(c["past"], 700)
        while c["requests"] * (c["past"] + c["new"]) * c["kv_heads"] * c["dim"] > 1 << 25 and c["past"]:
            c["past"] //= 2
        c["new_least"] = min(c["new_least"], c["new"])
        return c
    c.update(group=rng.choice([1, 2, 4, 4, 5, 8]), cap=rng.choice([0.0, 0.0, 0.0, 30.0, 50.0]),
             window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]), slopes=rng.random() < 0.2)
    while (c["requests"] * c["new"] * c["group"] * c["kv_heads"] * (c["past"] + c["new"]) > 1 << 30 or
           c["requests"] * (c["past"] + c["new"]) * c["kv_heads"] * c["dim"] > 1 << 28):
        k = max(("requests", "new", "past"), key=lambda n: c[n] * (1 if n == "requests" else 0.25 if n == "new" else 0.02))
        c[k] = c[k] // 2 + (k == "new")
    c["new_least"] = min(c["new_least"], c["new"])
    return c


# ---- inputs -----------------------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _lengths(c):
    """The new tokens and the cached tokens of each request, on the host: spread over their ranges, the same for every seed."""
    n, least = c["requests"], c["new_least"]
    spread = lambda i, k: (0.5 + (i + 1) * k) % 1.0  # noqa: E731
    new = [c["new"] if i == 0 else least + int((c["new"] + 1 - least) * spread(i, 0.6180339887)) for i in range(n)]
    past = [c["past"] if i == n - 1 else int((c["past"] + 1) * spread(i, 0.7548776662)) for i in range(n)]
    return new, past


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _tables(g, c):
    """The step's requests: lengths, slots in any order, and block tables whose blocks lie anywhere in the cache."""
    new, past = _lengths(c)
    n, bs = c["requests"], c["block"]
    blocks = [-(-(a + b) // bs) for a, b in zip(new, past)]
    width, total = max(blocks), sum(blocks)
    ids = torch.randperm(total + 3, generator=g, device=DEV).to(torch.int32)
    nb = _ints(blocks)
    at = torch.cumsum(nb, 0) - nb
    col = torch.arange(width, device=DEV)
    table = torch.where(col < nb[:, None], ids[(at[:, None] + col).clamp(max=total - 1)], -1).to(torch.int32)
    slots = torch.randperm(n + 2, generator=g, device=DEV)[:n].to(torch.int32)
    pages = torch.full((n + 2, width), -1, dtype=torch.int32, device=DEV)
    pages[slots.long()] = table
    starts = torch.zeros(n + 1, dtype=torch.int32, device=DEV)
    starts[1:] = torch.cumsum(_ints(new), 0)
    return {"new": new, "past_": past, "tokens": sum(new), "most_new": max(new), "most_len": max(a + b for a, b in zip(new, past)),
            "count": _ints(new), "past": _ints(past), "slots": slots, "pages": pages, "starts": starts, "blocks": total + 3}


def _scale_of(amax, fmt):
    """The power of two that a block's largest value gets: the smallest 2^e, e >= LEAST, with amax <= QMAX * 2^e."""
    m, e = torch.frexp(amax)
    e = e - (9 if fmt == "e4m3" else 7) + (m > QMAX[fmt] / (512 if fmt == "e4m3" else 128))
    e = torch.where(amax > 0, e, LEAST).clamp(min=LEAST)
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _codes(v, fmt):
    """Values in steps of their scale, rounded to codes (ties to even)."""
    if fmt == "e4m3":
        return v.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
    return v.round().clamp(-127.0, 127.0).to(torch.int8).view(torch.uint8)


def _values(codes, fmt):
    return codes.view(torch.float8_e4m3fn if fmt == "e4m3" else torch.int8).float()


def _cache(g, c, blocks):
    """A cache whose blocks are full: normal values with a size of its own for each block and head."""
    hk, bs, d = c["kv_heads"], c["block"], c["dim"]
    out = []
    for shape in ((blocks, hk, bs, d), (blocks, hk, bs // 16, d, 16)):
        size = torch.rand((blocks, hk), generator=g, device=DEV).mul_(1.5).add_(0.5)
        codes = torch.empty(shape, dtype=torch.uint8, device=DEV)
        scale = torch.empty((blocks, hk), device=DEV)
        step = max(1, (1 << 27) // (hk * bs * d))
        for i in range(0, blocks, step):
            v = torch.randn(codes[i:i + step].shape, generator=g, device=DEV)
            ones = (-1,) + (1,) * (len(shape) - 2)
            v *= size[i:i + step].reshape(v.shape[:2] + ones[1:])
            s = _scale_of(v.abs().flatten(2).amax(-1), c["format"])
            scale[i:i + step] = s
            codes[i:i + step] = _codes(v / s.reshape(v.shape[:2] + ones[1:]), c["format"])
        out += [codes, scale]
    return out


def prepare(case, seed):
    g, c = _gen(seed), case
    s = _tables(g, c)
    s["case"] = c
    if c["op"] == "pages":
        # before the step: the blocks of the new tokens are still in the free list, under others
        bs = c["block"]
        held = (s["past"] + bs - 1) // bs
        col = torch.arange(s["pages"].shape[1], device=DEV)
        spare = torch.randperm(s["blocks"] + 40, generator=g, device=DEV).to(torch.int32) + s["blocks"]
        rows = s["slots"].long()
        s["pages"][rows] = torch.where(col < held[:, None], s["pages"][rows], -1)
        need = [-(-(a + b) // bs) - -(-b // bs) for a, b in zip(s["new"], s["past_"])]
        s["free"] = spare[:sum(need) + 17].contiguous()
        s["n_free"] = _ints([len(s["free"]) - 5])
        s["rows"] = s["tokens"] + 13  # the step's arrays are longer than the step
        s["out"] = {"pages": s["pages"].clone(), "n_free": torch.zeros_like(s["n_free"]),
                    "starts": torch.zeros_like(s["starts"]), "seq": _ints([[0] * 4]).repeat(s["rows"], 1), "pos": _ints([0] * s["rows"])}
        return s
    s["k_codes"], s["k_scale"], s["v_codes"], s["v_scale"] = _cache(g, c, s["blocks"])
    t, hk, d = s["tokens"], c["kv_heads"], c["dim"]
    if c["op"] == "write":
        # K and V as the projections and rope leave them: V a view of a wider row
        s["k"] = torch.randn((t, hk, d), generator=g, device=DEV).to(TORCH[c["dtype"]])
        s["kv"] = torch.randn((t, 2, hk, d), generator=g, device=DEV).to(TORCH[c["dtype"]])
        s["v"] = s["kv"][:, 1]
        return s
    h = hk * c["group"]
    s["q"] = torch.randn((t, h, d), generator=g, device=DEV).to(TORCH[c["dtype"]])
    s["slopes"] = torch.rand(h, generator=g, device=DEV).mul_(0.05).add_(1e-4) if c["slopes"] else None
    s["y"] = torch.empty_like(s["q"])
    s["work"] = torch.empty(160 << 20, dtype=torch.uint8, device=DEV)
    return s


# ---- one pass ---------------------------------------------------------------------------------------------

def run(state):
    return globals()["_" + ("own" if own else "plain") + "_" + state["case"]["op"]](state, state["case"])


def _batch(s, native):
    return native.kv8_batch(s["case"]["requests"], s["tokens"], s["starts"].data_ptr(), s["past"].data_ptr(),
                            s["pages"].data_ptr(), s["pages"].shape[0], s["pages"].shape[1], slots=s["slots"].data_ptr())


def _cache_of(s, native):
    c = s["case"]
    return native.kv8_cache(c["format"], s["k_codes"].data_ptr(), s["v_codes"].data_ptr(), s["k_scale"].data_ptr(),
                            s["v_scale"].data_ptr(), s["blocks"], c["block"], c["kv_heads"], c["dim"])


def _own_pages(s, c):
    from sharplight_amd import native
    o = s["out"]
    if "call" not in s:  # the arguments' struct, which a program keeps with its buffers
        s["call"] = native.kv_pages(c["requests"], s["past"].data_ptr(), s["count"].data_ptr(), o["pages"].data_ptr(),
                                    o["pages"].shape[0], o["pages"].shape[1], c["block"], s["free"].data_ptr(), len(s["free"]),
                                    s["n_free"].data_ptr(), o["n_free"].data_ptr(), s["rows"], o["starts"].data_ptr(),
                                    seq=o["seq"].data_ptr(), pos=o["pos"].data_ptr(), slots=s["slots"].data_ptr())
    native.kv_pages_advance(s["call"])
    return [o["pages"], o["n_free"], o["starts"], o["seq"], o["pos"]]


def _own_write(s, c):
    from sharplight_amd import native
    if "call" not in s:
        s["call"] = _cache_of(s, native), _batch(s, native)
    hk, d = c["kv_heads"], c["dim"]
    native.kv8_write(c["dtype"], s["k"].data_ptr(), s["v"].data_ptr(), *s["call"], v_stride_t=2 * hk * d)
    return _cache_out(s, c)


def _own_attention(s, c):
    from sharplight_amd import native
    if "call" not in s:
        s["call"] = _cache_of(s, native), _batch(s, native)
    native.kv8_attention(c["dtype"], s["q"].data_ptr(), s["y"].data_ptr(), c["kv_heads"] * c["group"], *s["call"],
                         scale=1.0 / math.sqrt(c["dim"]), softcap=c["cap"], window=c["window"],
                         slopes=None if s["slopes"] is None else s["slopes"].data_ptr(), max_new=s["most_new"],
                         work=s["work"].data_ptr(), work_bytes=s["work"].numel())
    return s["y"]


def _cache_out(s, c):
    """The cache in its own 8-bit type, whose values count steps of the scales beside them."""
    kind = torch.float8_e4m3fn if c["format"] == "e4m3" else torch.int8
    return [s["k_codes"].view(kind), s["k_scale"], s["v_codes"].view(kind), s["v_scale"]]


def _rows_of(starts, past, tokens):
    """The request, the place in it and the position of each of the step's rows."""
    t = torch.arange(tokens, device=DEV, dtype=torch.int32)
    req = torch.searchsorted(starts, t, right=True) - 1
    at = t - starts[req]
    return req, at, past[req] + at


def _plain_pages(s, c):
    bs, past, count, rows = c["block"], s["past"], s["count"], s["rows"]
    pages = s["out"]["pages"].copy_(s["pages"])
    starts = s["out"]["starts"]
    starts[1:] = torch.cumsum(count, 0)
    held = (past + bs - 1) // bs
    need = (past + count + bs - 1) // bs - held
    before = torch.cumsum(need, 0) - need
    col = torch.arange(pages.shape[1], device=DEV)
    j = col - held[:, None]
    taken = s["free"][(s["n_free"] - 1 - (before[:, None] + j)).clamp(0, len(s["free"]) - 1)]
    table = torch.where((j >= 0) & (j < need[:, None]), taken, pages[s["slots"].long()])
    pages[s["slots"].long()] = table
    t = torch.arange(rows, device=DEV, dtype=torch.int32)
    there = t < starts[-1]
    req = (torch.searchsorted(starts, t, right=True) - 1).clamp(max=c["requests"] - 1)
    pos = past[req] + t - starts[req]
    block = table[req, (pos // bs).clamp(0, pages.shape[1] - 1)]
    seq = torch.stack([s["slots"][req], pos, req.to(torch.int32), block], 1)
    return [pages, s["n_free"] - need.sum().to(torch.int32), starts, torch.where(there[:, None], seq, -1), torch.where(there, pos, 0)]


def _plain_write(s, c):
    bs, fmt = c["block"], c["format"]
    req, _, pos = _rows_of(s["starts"], s["past"], s["tokens"])
    block = s["pages"][s["slots"][req].long(), pos // bs].long()
    off = (pos % bs).long()
    begun = torch.zeros(s["blocks"], dtype=torch.int32, device=DEV).index_reduce_(0, block, (off == 0).to(torch.int32) + 1, "amax")
    touched, fresh = begun > 0, begun > 1
    for x, codes, scale in ((s["k"], s["k_codes"], s["k_scale"]), (s["v"], s["v_codes"], s["v_scale"])):
        x = x.float()
        amax = torch.zeros_like(scale).index_reduce_(0, block, x.abs().amax(-1), "amax")
        s1 = torch.maximum(_scale_of(amax, fmt), torch.where(fresh[:, None], 0.0, scale))
        s1 = torch.where(touched[:, None], s1, scale)
        ones = (slice(None), slice(None)) + (None,) * (codes.dim() - 2)
        old = _codes(_values(codes, fmt) * (scale / s1)[ones], fmt)
        old = torch.where(fresh[(slice(None),) + (None,) * (codes.dim() - 1)], torch.zeros_like(old), old)
        fill = _codes(x / s1[block][:, :, None], fmt)
        if codes.dim() == 4:
            old[block, :, off] = fill
        else:
            old[block, :, off // 16, :, off % 16] = fill
        codes.copy_(old)
        scale.copy_(s1)
    return _cache_out(s, c)


def _plain_attention(s, c):
    n, hk, gr, d, bs, fmt = c["requests"], c["kv_heads"], c["group"], c["dim"], c["block"], c["format"]
    new, keys = s["most_new"], -(-s["most_len"] // bs) * bs
    table = s["pages"][s["slots"].long(), :keys // bs].clamp(min=0).long()
    k = _values(s["k_codes"][table], fmt) * s["k_scale"][table][..., None, None]
    k = k.permute(0, 2, 4, 1, 3).reshape(n * hk, d, keys)
    v = _values(s["v_codes"][table], fmt) * s["v_scale"][table][..., None, None, None]
    v = v.permute(0, 2, 1, 3, 5, 4).reshape(n * hk, keys, d)
    at = torch.arange(new, device=DEV)
    q = s["q"][(s["starts"][:-1, None] + at).clamp(max=s["tokens"] - 1).long()].float()
    q = q.reshape(n, new, hk, gr, d).permute(0, 2, 3, 1, 4).reshape(n * hk, gr * new, d)
    p = torch.bmm(q, k).reshape(n, hk, gr, new, keys).mul_(1.0 / math.sqrt(d))
    if c["cap"]:
        p = p.div_(c["cap"]).tanh_().mul_(c["cap"])
    far = torch.arange(keys, device=DEV) - (s["past"][:, None] + at)[:, :, None]  # [n, new, keys]: 0 at the row's own position
    if c["slopes"]:
        p += s["slopes"].reshape(1, hk, gr, 1, 1) * far[:, None, None].float()
    hide = far > 0
    if c["window"]:
        hide |= far <= -c["window"]
    p.masked_fill_(hide[:, None, None], -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    p = p.div_(p.sum(-1, keepdim=True)).reshape(n * hk, gr * new, keys)
    o = torch.bmm(p, v).reshape(n, hk, gr, new, d)
    req, place, _ = _rows_of(s["starts"], s["past"], s["tokens"])
    s["y"].copy_(o[req, :, :, place.long()].reshape(s["tokens"], hk * gr, d))
    return s["y"]


# ---- what a pass cannot do without ---------------------------------------------------------------------------

def work(case):
    c = case
    new, past = _lengths(c)
    t, bs = sum(new), c["block"]
    if c["op"] == "pages":
        taken = sum(-(-(a + b) // bs) - -(-b // bs) for a, b in zip(new, past))
        return {"bytes": 16 * len(new) + 20 * t + 8 * taken, "flops": 4 * t}
    per = c["kv_heads"] * c["dim"]
    if c["op"] == "write":
        touched = sum((a + b - 1) // bs - b // bs + 1 for a, b in zip(new, past))
        return {"bytes": 2 * t * per * (SIZE[c["dtype"]] + 1) + 16 * touched * c["kv_heads"], "flops": 4 * t * per}
    w = c["window"]
    seen = [min(a + b, w + a - 1) if w else a + b for a, b in zip(new, past)]  # keys that some row of the request sees
    if w:
        pairs = sum(sum(min(b + i + 1, w) for i in range(a)) for a, b in zip(new, past))
    else:
        pairs = sum(a * b + a * (a + 1) // 2 for a, b in zip(new, past))
    return {"bytes": 2 * per * sum(seen) + 2 * t * per * c["group"] * SIZE[c["dtype"]] + 8 * c["kv_heads"] * sum(-(-x // bs) for x in seen),
            "flops": 4 * per * c["group"] * pairs}


# ---- 64-bit reference ---------------------------------------------------------------------------------------

def _table_64(fmt):
    """What each of the 256 codes stands for."""
    out = []
    for b in range(256):
        if fmt == "i8":
            out.append(float(b - 256 if b > 127 else b))
            continue
        e, m = (b >> 3) & 15, b & 7
        v = math.nan if e == 15 and m == 7 else m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        out.append(-v if b > 127 else v)
    return torch.tensor(out, dtype=torch.float64, device=DEV)


def _power_64(e):
    """2^e of whole numbers e in 64 bits, exactly (a device's pow may be off in the last bit, which would break ties)."""
    return torch.tensor([2.0 ** k for k in range(-64, 129)], dtype=torch.float64, device=DEV)[e.long() + 64]


def _round_64(v, fmt):
    """v to the nearest value that a code stands for, ties to the even code."""
    if fmt == "i8":
        return torch.round(v)
    step = _power_64(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(v / step) * step


def exact(case, seed):
    c = case
    if c["op"] == "pages":
        return None  # whole numbers only
    s = prepare(c, seed)
    new, past = s["new"], s["past_"]
    pages, slots = s["pages"].tolist(), s["slots"].tolist()
    tab = _table_64(c["format"])
    return (_exact_write if c["op"] == "write" else _exact_attention)(s, c, new, past, pages, slots, tab)


def _exact_write(s, c, new, past, pages, slots, tab):
    bs, fmt, qmax = c["block"], c["format"], QMAX[c["format"]]
    out = []
    for x, codes, scale in ((s["k"], s["k_codes"], s["k_scale"]), (s["v"], s["v_codes"], s["v_scale"])):
        q = tab[codes.long()]
        if q.dim() == 5:  # V's codes as [blocks, heads, block, D]
            q = q.transpose(3, 4).flatten(2, 3).contiguous()
        sc = scale.double()
        x = x.double()
        first = 0
        for i, (a, b) in enumerate(zip(new, past)):
            for j in range(b // bs, (a + b - 1) // bs + 1):
                lo, hi = max(j * bs, b), min((j + 1) * bs, a + b)
                part = x[first + lo - b:first + hi - b].transpose(0, 1)  # [heads, tokens, D]
                block = pages[slots[i]][j]
                top = part.abs().amax((1, 2))
                s1 = _power_64(torch.ceil(torch.log2((top / qmax).clamp(min=2.0 ** LEAST))))
                if lo == j * bs:
                    q[block] = 0
                else:
                    s1 = torch.maximum(s1, sc[block])
                    q[block] = _round_64(q[block] * (sc[block] / s1)[:, None, None], fmt)
                q[block, :, lo - j * bs:hi - j * bs] = _round_64(part / s1[:, None, None], fmt)
                sc[block] = s1
            first += a
        if codes.dim() == 5:
            q = q.unflatten(2, (bs // 16, 16)).transpose(3, 4)
        out += [q.reshape(codes.shape), sc]
    return out


def _exact_attention(s, c, new, past, pages, slots, tab):
    hk, gr, d, bs = c["kv_heads"], c["group"], c["dim"], c["block"]
    y = torch.empty((s["tokens"], hk, gr, d), dtype=torch.float64, device=DEV)
    q = s["q"].double().reshape(s["tokens"], hk, gr, d)
    first = 0
    for i, (a, b) in enumerate(zip(new, past)):
        n = a + b
        ids = torch.tensor(pages[slots[i]][:-(-n // bs)], device=DEV)
        for h in range(hk):
            k = tab[s["k_codes"][ids, h].long()] * s["k_scale"][ids, h].double()[:, None, None]
            v = tab[s["v_codes"][ids, h].long()] * s["v_scale"][ids, h].double()[:, None, None, None]
            k = k.reshape(-1, d)[:n]
            v = v.transpose(2, 3).reshape(-1, d)[:n]
            step = max(1, (1 << 26) // (n * gr))
            for r in range(0, a, step):
                m = min(step, a - r)
                z = (q[first + r:first + r + m, h].reshape(m * gr, d) @ k.T).reshape(m, gr, n) / math.sqrt(d)
                if c["cap"]:
                    z = c["cap"] * torch.tanh(z / c["cap"])
                gap = torch.arange(n, device=DEV)[None] - (b + r + torch.arange(m, device=DEV))[:, None]
                if c["slopes"]:
                    z = z + s["slopes"].double().reshape(hk, gr)[h][None, :, None] * gap[:, None].double()
                see = gap <= 0
                if c["window"]:
                    see &= gap > -c["window"]
                z = torch.where(see[:, None], z, torch.full_like(z, -math.inf))
                w = torch.softmax(z, -1)
                y[first + r:first + r + m, h] = (w.reshape(m * gr, n) @ v).reshape(m, gr, d)
        first += a
    return y.reshape(s["tokens"], hk * gr, d)
