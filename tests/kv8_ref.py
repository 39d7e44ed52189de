"""Plain 64-bit statements of the paged 8-bit cache's operators (slhip_kv_pages_*, slhip_kv8_write, slhip_kv8_attention),
request by request, and how far the library's results may be from them."""
from __future__ import annotations

import numpy as np

QMAX = {"i8": 127.0, "e4m3": 448.0}


def code_values(fmt: str) -> np.ndarray:
    """What each of the 256 codes stands for."""
    b = np.arange(256)
    if fmt == "i8":
        return b.astype(np.uint8).view(np.int8).astype(np.float64)
    e, m = (b >> 3) & 15, b & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v = np.where(b > 127, -v, v)
    v[(b & 127) == 127] = np.nan
    return v


def to_codes(v: np.ndarray, fmt: str) -> np.ndarray:
    """Values in steps of their scale (|v| <= QMAX) to codes, rounded to nearest, ties to the even code. E4M3 zeros keep the
    sign of a negative value (code 0x80 stands for -0, the same value); -0 itself becomes +0."""
    if fmt == "i8":
        return np.rint(v).astype(np.int8).view(np.uint8)
    t = code_values("e4m3")[:127]  # 0 .. 448, increasing
    a = np.abs(v)
    hi = np.clip(np.searchsorted(t, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    up = (t[hi] - a < a - t[lo]) | ((t[hi] - a == a - t[lo]) & (hi % 2 == 0))
    c = np.where(up, hi, lo)
    return np.where(v < 0, c + 128, c).astype(np.uint8)


def scale_of(amax: float, fmt: str) -> np.float32:
    if not np.isfinite(amax) or amax > QMAX[fmt] * 2.0 ** 40:
        return np.float32(np.nan)
    e = -40
    while amax > QMAX[fmt] * 2.0 ** e:
        e += 1
    return np.float32(2.0 ** e)


class Cache:
    """Codes [blocks, heads, block_size, D] of K and [blocks, heads, block_size / 16, D, 16] of V, scales [blocks, heads]."""

    def __init__(self, fmt, blocks, bs, heads, D, fill=None):
        self.fmt, self.blocks, self.bs, self.heads, self.D = fmt, blocks, bs, heads, D
        shape = (blocks, heads, bs, D)
        if fill is None:
            self.k, self.v = np.zeros(shape, np.uint8), np.zeros((blocks, heads, bs // 16, D, 16), np.uint8)
            self.ks, self.vs = np.full((blocks, heads), 2.0 ** -40, np.float32), np.full((blocks, heads), 2.0 ** -40, np.float32)
        else:  # random codes and scales
            top = 255 if fmt == "i8" else 127
            self.k = fill.integers(0, top, shape).astype(np.uint8)
            self.v = fill.integers(0, top, (blocks, heads, bs // 16, D, 16)).astype(np.uint8)
            if fmt == "e4m3":  # values of a size: leave the largest exponents out, add signs
                self.k = (self.k % 104 | fill.integers(0, 2, shape) << 7).astype(np.uint8)
                self.v = (self.v % 104 | fill.integers(0, 2, self.v.shape) << 7).astype(np.uint8)
            s = lambda: (2.0 ** fill.integers(-9, -5, (blocks, heads))).astype(np.float32)  # noqa: E731
            self.ks, self.vs = s(), s()

    def copy(self):
        c = Cache.__new__(Cache)
        c.__dict__ = {k: v.copy() if isinstance(v, np.ndarray) else v for k, v in self.__dict__.items()}
        return c

    def keys(self, ids, h):
        """K and V of a request's blocks as values, [tokens, D] each, and V's scale a token."""
        t = code_values(self.fmt)
        k = t[self.k[ids, h]].reshape(-1, self.D)
        v = t[self.v[ids, h]].transpose(0, 1, 3, 2).reshape(-1, self.D)
        ks, vs = (np.repeat(s[ids, h].astype(np.float64), self.bs)[:, None] for s in (self.ks, self.vs))
        return k * ks, v * vs


def write(cache: Cache, k, v, starts, past, slots, pages):
    """slhip_kv8_write: k, v [T, heads, D] in f64. Requests that do not fit, and blocks outside the cache, are skipped."""
    tab, bs, fmt = code_values(cache.fmt), cache.bs, cache.fmt
    for i in range(len(past)):
        s0, s1, p, slot = int(starts[i]), int(starts[i + 1]), int(past[i]), int(slots[i])
        n = s1 - s0
        if not (0 <= s0 <= s1 <= len(k) and p >= 0 and 0 <= slot < len(pages) and p + n <= pages.shape[1] * bs):
            continue
        for j in range(p // bs, (p + n - 1) // bs + 1 if n else 0):
            block = int(pages[slot, j])
            if not 0 <= block < cache.blocks:
                continue
            lo, hi = max(j * bs, p), min((j + 1) * bs, p + n)
            for x, codes, scales in ((k, cache.k, cache.ks), (v, cache.v, cache.vs)):
                for h in range(cache.heads):
                    new = x[s0 + lo - p:s0 + hi - p, h]  # [tokens, D]
                    old = codes[block, h]
                    if codes.ndim == 5:  # as [tokens, D]
                        old = old.transpose(0, 2, 1).reshape(bs, cache.D)
                    old = old.copy()
                    with np.errstate(invalid="ignore"):
                        sn = scale_of(np.abs(new).max() if not np.isnan(new).any() else np.nan, fmt)
                    begun = lo == j * bs
                    s0_ = np.float32(0) if begun else scales[block, h]
                    s1_ = np.float32(np.nan) if np.isnan(sn) or np.isnan(s0_) else max(s0_, sn)
                    if begun:
                        old[:] = 0
                    elif s1_ > s0_:
                        old[:] = to_codes(tab[old] * (float(s0_) / float(s1_)), fmt)
                    old[lo - j * bs:hi - j * bs] = 0 if np.isnan(s1_) else to_codes(new / float(s1_), fmt)
                    codes[block, h] = old.reshape(bs // 16, 16, cache.D).transpose(0, 2, 1) if codes.ndim == 5 else old
                    scales[block, h] = s1_


def attention(cache: Cache, q, starts, past, slots, pages, *, scale, softcap=0.0, window=0, slopes=None, dtype="f32"):
    """slhip_kv8_attention in 64 bits: (y, bound), NaN rows where a row is not computed; q [T, H, D] in f64.

    bound: what an implementation with 32-bit sums and the header's roundings may be off, for each value of y. A weight
    w_j = softmax(z)_j is off by at most twice the largest error of a z (numerator and sum) relative to itself, so y by
    that times A = sum_j w_j |v_j|. The error of z_j:
      * the product: 2^-22 of sum_d |q_d k_d| for q's two f16 parts (bf16 rows are exact down to 2^-40 of the row's largest
        value a value: 2^-40 max|q| sum_d |k_d|, counted for both), and D 2^-24 of it for D sums in f32 in any order;
      * a cap: tanh to 2^-22 of the cap (its derivative is at most 1);
      * the exponent z log2(e) + log2(vs) - M and a slope's term: four roundings of 2^-24 of the largest magnitude;
      * 2^-22 for the exponential itself.
    The weights' rounding to f16: 2^-11 for bf16 activations (2^-33 of the largest contribution below that), 2^-22 for f32;
    sums over n keys and of partial sums: (n + 8) 2^-24 of A, in the numerator and in l. The output: 2^-8 (bf16), 2^-24 (f32)."""
    T, H, D = q.shape
    G = H // cache.heads
    y, bound = np.full(q.shape, np.nan), np.full(q.shape, np.nan)
    for i in range(len(past)):
        s0, s1, p, slot = int(starts[i]), int(starts[i + 1]), int(past[i]), int(slots[i])
        n = s1 - s0
        if not (0 <= s0 <= s1 <= T and p >= 0 and 0 <= slot < len(pages) and p + n <= pages.shape[1] * cache.bs):
            continue
        ids = pages[slot, :-(-(p + n) // cache.bs)]
        there = np.repeat((ids >= 0) & (ids < cache.blocks), cache.bs)[:p + n]
        ids = np.where((ids >= 0) & (ids < cache.blocks), ids, 0)
        for h in range(cache.heads):
            k, v = (x[:p + n] for x in cache.keys(ids, h))
            with np.errstate(divide="ignore", invalid="ignore"):
                lvs = np.log2(np.repeat(cache.vs[ids, h].astype(np.float64), cache.bs)[:p + n])
            for g in range(G):
                hq = h * G + g
                qq = q[s0:s1, hq]
                pos = p + np.arange(n)[:, None]
                gap = np.arange(p + n)[None] - pos
                see = (gap <= 0) & there[None]
                if window:
                    see &= gap > -window
                with np.errstate(invalid="ignore", over="ignore"):
                    z = scale * (qq @ k.T)
                    mag = abs(scale) * (np.abs(qq) @ np.abs(k).T)
                    dz = (2.0 ** -22 + D * 2.0 ** -24) * mag
                    dz += abs(scale) * 2.0 ** -40 * np.abs(qq).max(1, initial=0)[:, None] * np.abs(k).sum(1)[None]
                    if softcap:
                        z = softcap * np.tanh(z / softcap)
                        dz += 2.0 ** -22 * softcap
                    size = np.abs(z) * 1.4427 + np.abs(lvs)[None]
                    if slopes is not None:
                        z = z + slopes[hq] * gap
                        size = size + 1.4427 * np.abs(slopes[hq] * gap)
                    size = np.where(see, size, 0).max(1, initial=0)[:, None]
                    dz += 4 * 2.0 ** -24 * (2 * size + 16) + 2.0 ** -22
                    z = np.where(see, z, -np.inf)
                    m = z.max(1, keepdims=True, initial=-1e300)
                    w = np.exp(z - m)
                    l = w.sum(1, keepdims=True)
                    w = np.where(l > 0, w / np.where(l > 0, l, 1), 0)
                    w = np.where(see, w, 0)
                    vv = np.where(see.any(0)[:, None], v, 0)
                    y[s0:s1, hq] = w @ vv
                    A = w @ np.abs(vv)
                    top = (w[:, :, None] * np.abs(vv)[None]).max((1, 2), initial=0)[:, None] if n * (p + n) * D < 1 << 24 else A.max(1, keepdims=True)
                    wr = 2.0 ** -11 if dtype == "bf16" else 2.0 ** -22
                    err = 2 * np.where(see, dz, 0).max(1, initial=0)[:, None] + wr + 2 * (p + n + 8) * 2.0 ** -24
                    b = A * err + (p + n) * 2.0 ** -33 * (448.0 if cache.fmt == "e4m3" else 127.0) * top
                    bound[s0:s1, hq] = b * 1.01 + (2.0 ** -8 if dtype == "bf16" else 2.0 ** -24) * (np.abs(y[s0:s1, hq]) + b)
    return y, bound


def advance(past, count, slots, pages, bs, free, n_free, tokens):
    """slhip_kv_pages_advance: (ok, pages, n_free, starts, seq, pos)."""
    B = len(past)
    pages = pages.copy()
    bad = (len(set(map(int, slots))) < B or any(p < 0 or c < 0 or p + c > pages.shape[1] * bs for p, c in zip(past, count))
           or any(not 0 <= s < len(pages) for s in slots) or not 0 <= n_free <= len(free))
    starts, seq, pos = np.zeros(B + 1, np.int32), np.full((tokens, 4), -1, np.int32), np.zeros(tokens, np.int32)
    if not bad:
        need = [-(-(int(p) + int(c)) // bs) - -(-int(p) // bs) for p, c in zip(past, count)]
        bad = sum(need) > n_free or sum(map(int, count)) > tokens
    if bad:
        return False, pages, n_free, starts, seq, pos
    t = top = 0
    for i in range(B):
        held = -(-int(past[i]) // bs)
        for j in range(need[i]):
            pages[slots[i], held + j] = free[n_free - 1 - top]
            top += 1
        for k in range(int(count[i])):
            at = int(past[i]) + k
            seq[t] = (slots[i], at, i, pages[slots[i], at // bs])
            pos[t] = at
            t += 1
        starts[i + 1] = t
    return True, pages, n_free - top, starts, seq, pos


def release(past, slots, pages, bs, free, n_free):
    """slhip_kv_pages_release: (ok, pages, free, n_free)."""
    pages, free = pages.copy(), free.copy()
    need = [-(-int(p) // bs) for p in past]
    if (len(set(map(int, slots))) < len(past) or any(p < 0 or p > pages.shape[1] * bs for p in past)
            or any(not 0 <= s < len(pages) for s in slots) or not 0 <= n_free <= len(free) or n_free + sum(need) > len(free)):
        return False, pages, free, n_free
    for i, s in enumerate(slots):
        for j in range(need[i]):
            free[n_free] = pages[s, j]
            pages[s, j] = -1
            n_free += 1
    return True, pages, free, n_free
