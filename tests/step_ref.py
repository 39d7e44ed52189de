"""Plain 64-bit statements of what differs from request to request in a serving step (slhip_lora, slhip_draft_verify,
slhip_kv_pages_trim), request by request, and how far the library's results may be from them."""
from __future__ import annotations

import numpy as np


# ---- adapters ------------------------------------------------------------------------------------------------------

def lora(x, add, a, b, starts, adapter, rank=None, scale=None, bf16_parts=False):
    """(y, bound) in f64 of slhip_lora before its last rounding; add None: 0. Rows that no request has are NaN.

    bound: sums of K products in f32, in any order, are off by K * 2^-24 of the sum of the products' sizes; h so far off and as
    two bf16 parts (bf16_parts) by 2^-17 of itself; its scale and the sum over the ranks and `add` by (R + 3) * 2^-24 of the sizes. (Second-order terms:
    the factor 1.01.)"""
    T, K = x.shape
    y = np.full((T, b.shape[1]), np.nan)
    bound = np.zeros_like(y)
    for i in range(len(adapter)):
        s0, s1 = int(starts[i]), int(starts[i + 1])
        base = add[s0:s1] if add is not None else np.zeros((s1 - s0, b.shape[1]))
        ad = int(adapter[i])
        y[s0:s1] = base
        if not 0 <= ad < len(a):
            continue
        r = a.shape[1] if rank is None else int(np.clip(rank[ad], 0, a.shape[1]))
        s = 1.0 if scale is None else float(scale[ad])
        A, Bm, xs = a[ad, :r], b[ad, :, :r], x[s0:s1]
        h = xs @ A.T
        size = abs(xs) @ abs(A).T
        y[s0:s1] += s * (h @ Bm.T)
        off = K * 2.0 ** -24 * size + (2.0 ** -17 if bf16_parts else 0.0) * abs(h)
        bound[s0:s1] = 1.01 * (abs(s) * (off @ abs(Bm).T + (r + 3) * 2.0 ** -24 * (abs(h) @ abs(Bm).T)) + 2.0 ** -23 * abs(base))
    return y, bound


def rounded_bound(y, bound, dtype):
    """What the rounding to the result's type (half a step) adds."""
    half = 2.0 ** -24 if dtype == "f32" else 2.0 ** -8
    return bound * (1 + half) + half * np.abs(y)


# ---- drafts --------------------------------------------------------------------------------------------------------

def probabilities(z, tau):
    """softmax(z / tau) in f64, or None where the row cannot be used."""
    if np.isnan(z).any() or (z == np.inf).any() or not (z > -np.inf).any() or np.isnan(tau):
        return None
    tau = min(max(float(tau), 2.0 ** -40), 2.0 ** 40)
    with np.errstate(over="ignore"):
        e = np.where(z > -np.inf, np.exp((z - z.max()) / tau), 0.0)
    return e / e.sum()


def verify(target, draft, starts, ids, accept, sample, stride, tau=None, tau_q=None, past=None):
    """(out, n_out, kept, dropped, logp, margin) of slhip_draft_verify. margin: how near a choice came to a random number, at the
    least (in probability); the library's own sums may be off by some 2^-24."""
    B, V = len(sample), target.shape[1]
    out, logp = np.full((B, stride), -1, np.int64), np.zeros((B, stride))
    n_out, kept, dropped = np.zeros(B, np.int64), np.zeros(B, np.int64), np.zeros(B, np.int64)
    margin = np.inf
    for i in range(B):
        s0, s1 = int(starts[i]), int(starts[i + 1])
        p0 = 0 if past is None else int(past[i])
        kept[i] = p0
        n = s1 - s0
        if n <= 0 or n > stride:
            continue
        t = 1.0 if tau is None else float(tau[i])
        tq = t if tau_q is None else float(tau_q[i])
        greedy = t <= 0
        for j in range(n):
            z = target[s0 + j]
            x = int(ids[s0 + j + 1]) if j < n - 1 else None
            p = probabilities(z, 1.0 if greedy else t)
            if p is None:
                out[i, j], logp[i, j] = -1, np.nan
                break
            known = x is not None and 0 <= x < V
            if greedy:
                token = int(np.argmax(z))
                good = known and x == token
            else:
                chosen = draft is None or tq <= 0
                q = None if x is None or chosen else probabilities(draft[s0 + j], tq)
                if x is not None and chosen:
                    q = np.zeros(V)
                    if known:
                        q[x] = 1.0
                good = known and q is not None and accept[s0 + j] * q[x] < p[x]
                if known and q is not None:
                    margin = min(margin, abs(accept[s0 + j] * q[x] - p[x]) / max(p[x], q[x], 1e-300))
                if not good:
                    w = p if q is None else np.maximum(p - q, 0.0)
                    if not w.sum() > 0:
                        w = p
                    c = np.cumsum(w)
                    r = max(float(sample[i]), 0.0) * c[-1]
                    token = int(np.searchsorted(c, r, side="right"))
                    last = int(np.nonzero(w)[0][-1])
                    if sample[i] < 1:
                        margin = min(margin, np.abs(c[w > 0] - r).min())
                    if sample[i] > 0:
                        margin = min(margin, r)
                    token = min(token, last)
            if good:
                token = x
            out[i, j] = token
            with np.errstate(divide="ignore"):
                logp[i, j] = np.log(p[token])
            if not good:
                break
        n_out[i] = j + 1
        kept[i] = p0 + j + 1
        dropped[i] = n - j - 1
    return out, n_out, kept, dropped, logp, margin


def logp_bound(target, tau, lp):
    """How far a log-probability may be off: the sum's terms e by (2 + |log2 e|) 2^-23 of themselves, their f32 sums by 18 * 2^-24, and the
    rounding of the result."""
    t = 1.0 if tau <= 0 else min(max(tau, 2.0 ** -40), 2.0 ** 40)
    y = np.where(target > -np.inf, (target - target.max()) / t * np.log2(np.e), -np.inf)
    y = y[y > -200]
    e = np.exp2(y)
    return float((e * (2 + np.abs(y))).sum() / e.sum()) * 2.0 ** -23 + 18 * 2.0 ** -24 + abs(lp) * 2.0 ** -23


# ---- block tables --------------------------------------------------------------------------------------------------

def trim(past, count, slots, pages, bs, free, n_free):
    """slhip_kv_pages_trim: (ok, pages, free, n_free)."""
    pages, free = pages.copy(), free.copy()
    bad = (len(set(map(int, slots))) < len(past) or any(p < 0 or c < 0 or int(p) + int(c) > pages.shape[1] * bs for p, c in zip(past, count))
           or any(not 0 <= s < len(pages) for s in slots) or not 0 <= n_free <= len(free))
    if bad:
        return False, pages, free, n_free
    back = [(int(s), k) for p, c, s in zip(past, count, slots) for k in range(-(-int(p) // bs), -(-(int(p) + int(c)) // bs))]
    if n_free + len(back) > len(free) or any(pages[s, k] < 0 for s, k in back):
        return False, pages, free, n_free
    for o, (s, k) in enumerate(back):
        free[n_free + len(back) - 1 - o] = pages[s, k]
        pages[s, k] = -1
    return True, pages, free, n_free + len(back)
