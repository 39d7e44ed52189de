"""Performance cases of what differs from request to request in a serving step: low-rank adapters beside a shared projection,
the verification of drafted tokens, and the step back of the block tables behind the ones that were refused.

``lora``: y = add + s_a B_a (A_a x) for rows whose requests have adapters a of their own (or none). ``draft_verify``: target
logits, drafted tokens, the logits that they were drawn from and uniform random numbers in; accepted tokens and one more, drawn
from what is left of the target's probabilities, out, each with the logarithm of its probability. ``kv_pages_trim``: requests give
the blocks behind their kept tokens back.
``run`` makes those calls where ``own`` is true; otherwise it computes the same from elementary torch operations. ``exact``
restates the adapters' sums and the tokens' probabilities in 64 bits; all else is whole numbers.

Ranges that ``draw`` covers: 1 to 512 requests; adapters of 1 to 128 ranks, 1 to 128 of them, projections of 64 to 14336 inputs and
outputs, odd ones among them, f32 and bf16 activations with f32, f16 and bf16 adapters, one token to prompts of 8192; vocabularies
of 1000 to 262144, up to 16 drafts a request, drawn or chosen, f32 and bf16 logits, masked or not, with greedy requests among
them; tables of up to 32768 tokens a request.
"""
import math

import torch

own = False

DEV = "cuda"
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one chat's next token through an adapter of rank 16, where latency is most of it
        {"name": "lora_one", "op": "lora", "requests": 1, "new": 1, "new_least": 1, "adapters": 8, "rank": 16, "ragged": False,
         "none": 0.0, "k": 4096, "n": 4096, "x": "bf16", "w": "bf16", "pad": 0},
        # a decode step of 64 sequences, an adapter each, into the wide projection
        {"name": "lora_decode", "op": "lora", "requests": 64, "new": 1, "new_least": 1, "adapters": 64, "rank": 16, "ragged": False,
         "none": 0.0, "k": 4096, "n": 14336, "x": "bf16", "w": "bf16", "pad": 0},
        # a larger batch that shares eight adapters of several ranks, some requests without one, in an f32 graph
        {"name": "lora_shared_f32", "op": "lora", "requests": 256, "new": 1, "new_least": 1, "adapters": 8, "rank": 64, "ragged": True,
         "none": 0.2, "k": 14336, "n": 4096, "x": "f32", "w": "bf16", "pad": 3},
        # a long prompt's wide projection
        {"name": "lora_prefill", "op": "lora", "requests": 1, "new": 8192, "new_least": 8192, "adapters": 4, "rank": 16, "ragged": False,
         "none": 0.0, "k": 4096, "n": 14336, "x": "bf16", "w": "bf16", "pad": 0},
        # ragged prompt chunks over f16 adapters, f32 activations, sizes off the grid
        {"name": "lora_chunks_f32", "op": "lora", "requests": 23, "new": 180, "new_least": 3, "adapters": 7, "rank": 24, "ragged": True,
         "none": 0.1, "k": 2880, "n": 4104, "x": "f32", "w": "f16", "pad": 5},
        # one chat's four drafted tokens, the smallest verification
        {"name": "verify_one", "op": "verify", "requests": 1, "new": 5, "new_least": 5, "vocab": 151936, "dtype": "f32", "drawn": True,
         "greedy": 0.0, "top": 0, "temperature": 0.8, "pad": 0},
        # a batch's drafts, three to five a request, against the draft model's own logits
        {"name": "verify_batch", "op": "verify", "requests": 64, "new": 5, "new_least": 3, "vocab": 151936, "dtype": "f32", "drawn": True,
         "greedy": 0.0, "top": 0, "temperature": 1.0, "pad": 0},
        # many requests' next tokens without drafts, bf16 logits of an odd vocabulary, greedy ones among them
        {"name": "sample_bf16", "op": "verify", "requests": 256, "new": 1, "new_least": 1, "vocab": 50257, "dtype": "bf16", "drawn": False,
         "greedy": 0.25, "top": 0, "temperature": 0.7, "pad": 0},
        # drafts looked up in the prompt (chosen, not drawn), against logits of which all but 50 a row are masked
        {"name": "verify_lookup", "op": "verify", "requests": 16, "new": 13, "new_least": 1, "vocab": 32000, "dtype": "f32", "drawn": False,
         "greedy": 0.2, "top": 50, "temperature": 1.0, "pad": 5},
        # a batch whose refused drafts end in blocks of their own now and then
        {"name": "trim_drafts", "op": "trim", "requests": 64, "new": 5, "new_least": 0, "past": 4096, "block": 16},
        # contexts cut back by hundreds of tokens each, as after a stopped generation
        {"name": "trim_long", "op": "trim", "requests": 333, "new": 2000, "new_least": 1, "past": 2048, "block": 32},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["lora", "lora", "lora", "verify", "verify", "verify", "trim"])
    if op == "trim":
        new = _log(rng, 1, 2000)
        c = {"op": op, "requests": _log(rng, 1, 512), "new": new, "new_least": _log(rng, 1, new) - 1, "past": _log(rng, 1, 30000) - 1,
             "block": rng.choice([16, 16, 32, 64, 128])}
        while c["requests"] * c["new"] > 1 << 20:
            c["requests"] = c["requests"] // 2 + 1
            c["new"] = c["new"] // 2 + 1
        c["new_least"] = min(c["new_least"], c["new"])
        return c
    if op == "verify":
        new = rng.choice([1, 1, 2, 3, 4, 5, 6, 8, 11, 17])
        c = {"op": op, "requests": _log(rng, 1, 512), "new": new, "new_least": rng.randint(1, new), "vocab": _log(rng, 1000, 262144),
             "dtype": rng.choice(["f32", "f32", "bf16"]), "drawn": rng.random() < 0.6, "greedy": rng.choice([0.0, 0.0, 0.25, 1.0]),
             "top": rng.choice([0, 0, 0, 40]), "temperature": rng.choice([0.5, 0.7, 1.0, 1.0, 1.3]), "pad": rng.choice([0, 0, 1, 8])}
        while c["requests"] * c["new"] * c["vocab"] > 300 * 151936:
            c["requests"] = c["requests"] // 2 + (c["requests"] == 1)
            if c["requests"] <= 2:
                c["vocab"] = c["vocab"] // 2 + 1
        return c
    new = 1 if rng.random() < 0.4 else _log(rng, 2, 8192)
    size = lambda: rng.choice([512, 1024, 2048, 2880, 4096, 5120, 8192, 14336, _log(rng, 64, 14336), 8 * _log(rng, 8, 1792)])  # noqa: E731
    c = {"op": op, "requests": _log(rng, 1, 512), "new": new, "new_least": _log(rng, 1, new), "adapters": _log(rng, 1, 128),
         "rank": rng.choice([1, 4, 8, 8, 16, 16, 16, 32, 64, 128, rng.randint(2, 100)]), "ragged": rng.random() < 0.4,
         "none": rng.choice([0.0, 0.0, 0.3]), "k": size(), "n": size(), "x": rng.choice(["bf16", "bf16", "f32"]),
         "w": rng.choice(["bf16", "bf16", "f16", "f32"]), "pad": rng.choice([0, 0, 7])}
    while c["requests"] * c["new"] * (c["k"] + c["n"]) > 8192 * 18432:
        big = max(("requests", "new"), key=lambda n: c[n] * (4 if n == "requests" else 1))
        c[big] = c[big] // 2 + 1
    # the plain form multiplies all rows by all adapters
    while c["adapters"] > 1 and c["requests"] * c["new"] * c["adapters"] * c["rank"] * (c["k"] + c["n"]) > 8192 * 64 * 18432:
        c["adapters"] //= 2
    while c["adapters"] * c["rank"] * (c["k"] + c["n"]) > 64 << 20:
        c["adapters"] //= 2
    c["new_least"] = min(c["new_least"], c["new"])
    return c


# ---- inputs -----------------------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _spread(i, k):
    return (0.5 + (i + 1) * k) % 1.0


def _rows(c):
    """The rows of each request, on the host: spread over their range, the same for every seed."""
    least = c["new_least"]
    return [c["new"] if i == 0 else least + int((c["new"] + 1 - least) * _spread(i, 0.6180339887)) for i in range(c["requests"])]


def _ranks(c):
    return [c["rank"] if i == 0 or not c["ragged"] else 1 + int(c["rank"] * _spread(i, 0.4142135623)) for i in range(c["adapters"])]


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _floats(v):
    return torch.tensor(v, dtype=torch.float32, device=DEV)


def _normal(g, shape, size, dtype):
    return torch.randn(shape, generator=g, device=DEV).mul_(size).to(dtype)


def prepare(case, seed):
    g, c = _gen(seed), case
    return {"case": c, **globals()["_prepare_" + c["op"]](g, c)}


def _prepare_lora(g, c):
    new = _rows(c)
    tokens, n_ad, r = sum(new) + c["pad"], c["adapters"], c["rank"]  # the step's arrays may be longer than the step
    starts = torch.zeros(c["requests"] + 1, dtype=torch.int32, device=DEV)
    starts[1:] = torch.cumsum(_ints(new), 0)
    order = torch.randperm(max(c["requests"], n_ad), generator=g, device=DEV)[:c["requests"]] % n_ad
    none = torch.rand(c["requests"], generator=g, device=DEV) < c["none"]
    t = TORCH[c["x"]]
    s = {"tokens": tokens, "new": new, "starts": starts, "adapter": torch.where(none, -1, order).to(torch.int32),
         "ranks": _ints(_ranks(c)), "scale": _floats([2.0 if i % 3 else 0.5 for i in range(n_ad)]),
         "x": _normal(g, (tokens, c["k"]), 1.0, t), "add": _normal(g, (tokens, c["n"]), 1.0, t)}
    s["a"] = _normal(g, (n_ad, r, c["k"]), c["k"] ** -0.5, TORCH[c["w"]])
    s["b"] = _normal(g, (n_ad, c["n"], r), 0.25 * r ** -0.5, TORCH[c["w"]])
    s["y"] = torch.zeros_like(s["add"])  # rows behind the last request's stay
    s["work"] = torch.empty(64 << 20, dtype=torch.uint8, device=DEV)
    return s


def _prepare_verify(g, c):
    new, v, dtype = _rows(c), c["vocab"], TORCH[c["dtype"]]
    n, tokens = c["requests"], sum(new)
    starts = torch.zeros(n + 1, dtype=torch.int32, device=DEV)
    starts[1:] = torch.cumsum(_ints(new), 0)
    # logits as a model's head leaves them: most far below a few high ones; the draft's are near the target's
    z = torch.randn((tokens, v + c["pad"]), generator=g, device=DEV).mul_(2.5)
    z[:, :v] += 6.0 * (torch.rand((tokens, v), generator=g, device=DEV) < 8.0 / v)
    tau = c["temperature"]
    greedy = (torch.arange(n, device=DEV) * 0.7548776662 + 0.3) % 1.0 < c["greedy"]
    s = {"tokens": tokens, "new": new, "starts": starts, "most": max(new),
         "temperature": torch.where(greedy, 0.0, tau * (0.8 + 0.4 * torch.rand(n, generator=g, device=DEV)))}
    near = z[:, :v] + 0.5 * torch.randn((tokens, v), generator=g, device=DEV)
    if c["drawn"]:  # the drafts: drawn from the draft's probabilities, as a draft model does
        draft = torch.zeros((tokens, v + c["pad"]), dtype=dtype, device=DEV)
        draft[:, :v] = near
        req = torch.searchsorted(starts, torch.arange(tokens, device=DEV, dtype=torch.int32), right=True) - 1
        heat = s["temperature"][req.clamp(max=n - 1)].clamp(min=1e-3)
        noise = torch.rand((tokens, v), generator=g, device=DEV).clamp_(min=1e-30).log_().neg_().log_()
        drafted = (draft[:, :v].float() / heat[:, None] - noise).argmax(-1)
        s["draft"] = draft
    else:  # or what stood in the prompt: mostly the likely one
        drafted = torch.where(torch.rand(tokens, generator=g, device=DEV) < 0.7, z[:, :v].argmax(-1), near.argmax(-1))
        s["draft"] = None
    if c["top"]:
        kept = z[:, :v].topk(min(c["top"], v), -1).values[:, -1:]
        z[:, :v] = torch.where(z[:, :v] < kept, -math.inf, z[:, :v])
    s["target"] = z.to(dtype)
    ids = torch.randint(0, v, (tokens,), generator=g, device=DEV, dtype=torch.int32)
    ids[1:] = drafted[:-1].to(torch.int32)  # row t's draft is the step's token t + 1
    s["ids"] = ids
    s["accept"] = torch.rand(tokens, generator=g, device=DEV)
    s["sample"] = torch.rand(n, generator=g, device=DEV)
    s["past"] = torch.randint(0, 4000, (n,), generator=g, device=DEV, dtype=torch.int32)
    s["out"] = {"tokens": _ints([0]).repeat(n, s["most"]), "n": _ints([0] * n), "kept": _ints([0] * n), "dropped": _ints([0] * n),
                "logp": _floats([0.0]).repeat(n, s["most"])}
    s["work"] = torch.empty(16 << 20, dtype=torch.uint8, device=DEV)
    return s


def _trim_lengths(c):
    n, least = c["requests"], c["new_least"]
    count = [c["new"] if i == 0 else least + int((c["new"] + 1 - least) * _spread(i, 0.6180339887)) for i in range(n)]
    past = [c["past"] if i == n - 1 else int((c["past"] + 1) * _spread(i, 0.7548776662)) for i in range(n)]
    return past, count


def _blocks(tokens, bs):
    return -(-tokens // bs)


def _prepare_trim(g, c):
    past, count = _trim_lengths(c)
    n, bs = c["requests"], c["block"]
    blocks = [_blocks(a + b, bs) for a, b in zip(past, count)]
    width, total = max(blocks + [1]), sum(blocks)
    back = total - sum(_blocks(a, bs) for a in past)
    ids = torch.randperm(total + 40, generator=g, device=DEV).to(torch.int32)
    nb = _ints(blocks)
    at = torch.cumsum(nb, 0) - nb
    col = torch.arange(width, device=DEV)
    table = torch.where(col < nb[:, None], ids[(at[:, None] + col).clamp(max=total + 39)], -1).to(torch.int32)
    slots = torch.randperm(n + 2, generator=g, device=DEV)[:n].to(torch.int32)
    before = torch.full((n + 2, width), -1, dtype=torch.int32, device=DEV)
    before[slots.long()] = table
    free = torch.full((back + 50,), -1, dtype=torch.int32, device=DEV)
    free[:40] = ids[total:]
    return {"past": _ints(past), "count": _ints(count), "slots": slots, "before": before, "free": free, "n_free": _ints([40]),
            "out": {"pages": before.clone(), "n_free": _ints([0])}}


# ---- one pass ---------------------------------------------------------------------------------------------

def run(state):
    return globals()["_" + ("own" if own else "plain") + "_" + state["case"]["op"]](state, state["case"])


def _own_lora(s, c):
    from sharplight_amd import native
    if "call" not in s:  # the arguments' structs, which a program keeps with its buffers
        s["call"] = (native.lora_set(c["w"], s["a"].data_ptr(), s["b"].data_ptr(), c["adapters"], c["rank"], c["k"], c["n"],
                                     rank=s["ranks"].data_ptr(), scale=s["scale"].data_ptr()),
                     native.lora_rows(c["requests"], s["tokens"], s["starts"].data_ptr(), s["adapter"].data_ptr()))
    native.lora(c["x"], c["x"], s["x"].data_ptr(), s["add"].data_ptr(), s["y"].data_ptr(), *s["call"], work=s["work"].data_ptr(),
                work_bytes=s["work"].numel())
    return s["y"]


def _plain_lora(s, c):
    # all adapters in one product each way; a row keeps the sums of its own
    n_ad, r = c["adapters"], c["rank"]
    t = torch.arange(s["tokens"], device=DEV, dtype=torch.int32)
    req = torch.searchsorted(s["starts"], t, right=True) - 1
    there = t < s["starts"][-1]
    mine = torch.where(there, s["adapter"][req.clamp(max=c["requests"] - 1)], -1)
    keep = (torch.arange(n_ad, device=DEV)[:, None] == mine[:, None, None]) & (torch.arange(r, device=DEV) < s["ranks"][:, None])
    h = (s["x"].float() @ s["a"].float().reshape(n_ad * r, c["k"]).T).reshape(-1, n_ad, r) * s["scale"][:, None]
    h = torch.where(keep, h, 0.0).reshape(-1, n_ad * r)
    y = h @ s["b"].float().transpose(0, 1).reshape(c["n"], n_ad * r).T + s["add"].float()
    s["y"].copy_(torch.where(there[:, None], y, 0.0))
    return s["y"]


def _own_verify(s, c):
    from sharplight_amd import native
    o = s["out"]
    if "call" not in s:
        s["call"] = native.drafts(c["requests"], s["tokens"], c["vocab"], s["starts"].data_ptr(), s["ids"].data_ptr(),
                                  s["accept"].data_ptr(), s["sample"].data_ptr(), o["tokens"].data_ptr(), s["most"], o["n"].data_ptr(),
                                  temperature=s["temperature"].data_ptr(), past=s["past"].data_ptr(), kept=o["kept"].data_ptr(),
                                  dropped=o["dropped"].data_ptr(), logp=o["logp"].data_ptr())
    native.draft_verify(c["dtype"], s["target"].data_ptr(), None if s["draft"] is None else s["draft"].data_ptr(), s["call"],
                        target_stride=c["vocab"] + c["pad"], draft_stride=c["vocab"] + c["pad"], work=s["work"].data_ptr(),
                        work_bytes=s["work"].numel())
    return [o["tokens"], o["n"], o["kept"], o["dropped"], o["logp"]]


def _plain_verify(s, c):
    v, n, most, starts = c["vocab"], c["requests"], s["most"], s["starts"].long()
    t = torch.arange(s["tokens"], device=DEV)
    req = torch.searchsorted(starts, t, right=True) - 1
    last = t == starts[req + 1] - 1
    tau = s["temperature"].double()[req][:, None]
    greedy = tau[:, 0] <= 0
    heat = torch.where(tau > 0, tau, 1.0)
    z = s["target"][:, :v].double()
    best = z.argmax(-1)
    top = z.amax(-1, keepdim=True)
    p = torch.exp((z - top) / heat)
    sums = p.sum(-1, keepdim=True)
    p /= sums
    x = torch.where(last, 0, s["ids"].roll(-1).long())
    if s["draft"] is None:
        q = torch.zeros_like(p).scatter_(1, x[:, None], 1.0)
    else:
        q = s["draft"][:, :v].double()
        q = torch.exp((q - q.amax(-1, keepdim=True)) / heat)
        q /= q.sum(-1, keepdim=True)
    px, qx = p.gather(1, x[:, None])[:, 0], q.gather(1, x[:, None])[:, 0]
    good = torch.where(greedy, x == best, s["accept"].double() * qx < px) & ~last
    place = torch.arange(most, device=DEV)
    rows = starts[:-1, None] + place
    some = rows < starts[1:, None]
    a = (good[rows.clamp(max=s["tokens"] - 1)] & some).long().cumprod(-1).sum(-1)  # accepted drafts of each request
    at = starts[:-1] + a
    w = torch.where(last[at, None], p[at], (p[at] - q[at]).clamp(min=0.0))
    total = torch.cumsum(w, -1)
    none = total[:, -1:] <= 0
    total = torch.where(none, torch.cumsum(p[at], -1), total)
    w = torch.where(none, p[at], w)
    drawn = (total <= s["sample"].double()[:, None] * total[:, -1:]).sum(-1)
    highest = torch.where(w > 0, torch.arange(v, device=DEV), -1).amax(-1)
    final = torch.where(greedy[at], best[at], torch.minimum(drawn, highest))
    row = rows.clamp(max=s["tokens"] - 1)
    out = torch.where(place < a[:, None], x[row], -1)
    out = torch.where(place == a[:, None], final[:, None], out)
    logp = (z[row, out.clamp(min=0)] - top[row, 0]) / heat[row, 0] - torch.log(sums[row, 0])
    o = s["out"]
    o["tokens"].copy_(out)
    o["logp"].copy_(torch.where(out >= 0, logp, 0.0))
    o["n"].copy_(a + 1)
    o["kept"].copy_(s["past"] + a + 1)
    o["dropped"].copy_(starts[1:] - starts[:-1] - a - 1)
    return [o["tokens"], o["n"], o["kept"], o["dropped"], o["logp"]]


def _own_trim(s, c):
    from sharplight_amd import native
    o = s["out"]
    if "call" not in s:
        s["call"] = native.kv_pages(c["requests"], s["past"].data_ptr(), s["count"].data_ptr(), o["pages"].data_ptr(),
                                    o["pages"].shape[0], o["pages"].shape[1], c["block"], s["free"].data_ptr(), len(s["free"]),
                                    s["n_free"].data_ptr(), o["n_free"].data_ptr(), slots=s["slots"].data_ptr())
    o["pages"].copy_(s["before"])  # the table as the step before left it
    native.kv_pages_trim(s["call"])
    return [o["pages"], o["n_free"], s["free"]]


def _plain_trim(s, c):
    bs, pages, free = c["block"], s["out"]["pages"], s["free"]
    pages.copy_(s["before"])
    keep = (s["past"] + bs - 1) // bs
    back = (s["past"] + s["count"] + bs - 1) // bs - keep
    before = torch.cumsum(back, 0) - back
    col = torch.arange(pages.shape[1], device=DEV)
    j = col - keep[:, None]
    goes = (j >= 0) & (j < back[:, None])
    table = pages[s["slots"].long()]
    n_free = s["n_free"] + back.sum()
    place = torch.where(goes, n_free - 1 - (before[:, None] + j), len(free))  # the first one goes on top
    padded = torch.cat([free, free[:1]]).scatter_(0, place.reshape(-1).long(), table.reshape(-1))
    free.copy_(padded[:-1])
    pages[s["slots"].long()] = torch.where(goes, -1, table)
    s["out"]["n_free"].copy_(n_free)
    return [pages, s["out"]["n_free"], free]


# ---- what a pass cannot do without ---------------------------------------------------------------------------

def work(case):
    c = case
    if c["op"] == "trim":
        past, count = _trim_lengths(c)
        back = sum(_blocks(a + b, c["block"]) - _blocks(a, c["block"]) for a, b in zip(past, count))
        return {"bytes": 12 * len(past) + 12 * back, "flops": 4 * len(past)}
    new = _rows(c)
    t = sum(new)
    if c["op"] == "verify":  # rows of greedy requests need no draft's logits, nor does a request's last row
        v, size = c["vocab"], SIZE[c["dtype"]]
        drafts = t - len(new) if c["drawn"] else 0
        return {"bytes": (t + (1 - c["greedy"]) * drafts) * v * size + 12 * t + 28 * len(new), "flops": 4 * t * v}
    ranks = _ranks(c)
    used = min(len(new) * (1 - c["none"]), c["adapters"])
    mean = sum(ranks) / len(ranks)
    rows = t * (1 - c["none"])
    return {"bytes": SIZE[c["x"]] * (rows * c["k"] + 2 * t * c["n"]) + SIZE[c["w"]] * used * mean * (c["k"] + c["n"]) + 8 * len(new),
            "flops": 2 * rows * mean * (c["k"] + c["n"])}


# ---- 64-bit reference ---------------------------------------------------------------------------------------

def exact(case, seed):
    if case["op"] == "trim":
        return None  # whole numbers only
    s, c = prepare(case, seed), case
    if case["op"] == "verify":
        return [None, None, None, None, _exact_logp(s, c)]
    y = torch.zeros((s["tokens"], c["n"]), dtype=torch.float64, device=DEV)
    ranks, scale = _ranks(c), s["scale"].tolist()
    first = 0
    for n, a in zip(s["new"], s["adapter"].tolist()):
        y[first:first + n] = s["add"][first:first + n].double()
        if a >= 0:
            h = s["x"][first:first + n].double() @ s["a"][a, :ranks[a]].double().T.contiguous()
            y[first:first + n] += scale[a] * (h @ s["b"][a, :, :ranks[a]].double().T.contiguous())
        first += n
    return y


def _exact_logp(s, c):
    """Request by request: its tokens, and the logarithms of their probabilities."""
    v = c["vocab"]
    out = torch.zeros((c["requests"], s["most"]), dtype=torch.float64, device=DEV)
    first = 0
    ids, accept, sample, heat = (s[k].tolist() for k in ("ids", "accept", "sample", "temperature"))
    for i, n in enumerate(s["new"]):
        tau = heat[i] if heat[i] > 0 else 1.0
        for j in range(n):
            row = s["target"][first + j, :v].double()
            lp = torch.log_softmax(row / tau, -1)
            x = ids[first + j + 1] if j < n - 1 else None
            if heat[i] <= 0:
                token = int(row.argmax())
            else:
                q = torch.zeros_like(lp)
                if x is not None and s["draft"] is None:
                    q[x] = 1.0
                elif x is not None:
                    q = torch.softmax(s["draft"][first + j, :v].double() / tau, -1)
                p = lp.exp()
                token = x
                if x is None or not accept[first + j] * float(q[x]) < float(p[x]):
                    w = (p - q).clamp(min=0.0)
                    sums = torch.cumsum(w if float(w.sum()) > 0 else p, -1)
                    token = min(int(torch.searchsorted(sums, sample[i] * sums[-1:], right=True)), v - 1)
            out[i, j] = lp[token]
            if token != x:
                break
        first += n
    return out
