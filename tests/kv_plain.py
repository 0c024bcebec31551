"""Caches of fp16 and fp32 rows in plain numpy: rows rotated and appended, a
draft's attention over them in float64 with a bound on what fp32 work may be off
by, and the walk that accepts drafted rows."""
from __future__ import annotations

import numpy as np

TYPES = {0: np.float32, 1: np.float16}


class Cache:
    """Host planes of one cache: contiguous (page = 0) or paged. What nothing was written to holds NaN."""

    def __init__(self, seqs, heads, d, cap, page=0, dtype=1, layers=1, seed=0):
        rng = np.random.default_rng(seed)
        self.seqs, self.heads, self.d, self.page, self.dtype, self.layers = seqs, heads, d, page, dtype, layers
        if page:
            self.per = -(-cap // page)
            self.s, self.rows = seqs * self.per + 2, page
            self.table = rng.permutation(self.s)[:seqs * self.per].reshape(seqs, self.per).astype(np.int32)
            self.cap = self.per * page
        else:
            self.per, self.s, self.rows, self.table, self.cap = 1, seqs, cap, None, cap
        self.planes = {w: np.full((layers, self.s, heads, self.rows, d), np.nan, TYPES[dtype]) for w in "kv"}

    def at(self, b, pos):
        """(plane, row) of a position, None where the cache has no such row."""
        if pos < 0 or pos >= self.cap:
            return None
        if self.table is None:
            return b, pos
        s = int(self.table[b, pos // self.page])
        return (s, pos % self.page) if 0 <= s < self.s else None

    def write(self, which, b, pos, x, layer=0):
        """x [heads, D] at position pos of sequence b."""
        at = self.at(b, pos)
        if at is not None:
            with np.errstate(over="ignore"):
                self.planes[which][layer, at[0], :, at[1]] = x

    def fill(self, lens, seed=1):
        rng = np.random.default_rng(seed)
        spread = np.exp(0.5 * rng.standard_normal((self.heads, self.d)))
        for layer in range(self.layers):
            for which in "kv":
                for b, n in enumerate(lens):
                    x = rng.standard_normal((max(int(n), 0), self.heads, self.d)) * (spread if which == "k" else 1.0)
                    for pos in range(len(x)):
                        self.write(which, b, pos, x[pos], layer)

    def rows_of(self, which, b, n, layer=0):
        """The values [heads, n, D] of the first n positions in float64, and which of them the cache has."""
        out = np.zeros((self.heads, n, self.d))
        has = np.zeros(n, bool)
        for pos in range(n):
            at = self.at(b, pos)
            if at is not None:
                has[pos] = True
                out[:, pos] = self.planes[which][layer, at[0], :, at[1]]
        return out, has


# ---- trees ---------------------------------------------------------------------------

def random_parents(rng, b, t, deep=False):
    """Trees [b, t]; deep: long lines."""
    p = np.full((b, t), -1, np.int32)
    for i in range(1, t):
        p[:, i] = i - 1 - rng.integers(0, min(i, 3), b) if deep else (rng.random(b) ** 2 * i).astype(np.int32)
    return p


def line(parents, t):
    """Row t and its ancestors, from t on; a number that is not an earlier row's ends it."""
    out = [t]
    while 0 <= parents[out[-1]] < out[-1]:
        out.append(int(parents[out[-1]]))
    return out


def chain(t):
    return np.arange(-1, t - 1, dtype=np.int32)


# ---- appended rows -------------------------------------------------------------------

def rotate(x, angle_pos, base, rot, interleaved, divisors):
    """x [..., D] float64 turned for position angle_pos -> (turned, bound).

    The bound: an angle, in 64 bits, is off by at most 2^-48 of itself (the exponential's argument, up to 20, the
    division and the products round 2^-53 of it each, 20 times), cosine and sine by 4 2^-24 (the angle rounded to fp32,
    the series' terms), a rotated value by those times its two values and 3 roundings of a product or sum."""
    y, bound = x.copy(), np.zeros(x.shape)
    i = np.arange(rot // 2)
    theta = angle_pos * float(np.float32(base)) ** (-2.0 * i / rot) if rot else np.zeros(0)
    if divisors is not None:
        d = divisors[:rot // 2].astype(np.float64)
        theta = np.where(d > 0, theta / np.where(d > 0, d, 1), theta)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    c, s = np.cos(theta), np.sin(theta)
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    off = (np.abs(x[..., a]) + np.abs(x[..., b])) * (np.abs(theta) * 2.0 ** -48 + 7 * 2.0 ** -24)
    bound[..., a] = bound[..., b] = off
    return y, bound


def append(cache, q, k, v, positions, counts=None, angles=None, base=1e4, rot=None, interleaved=False, divisors=None, layer=0):
    """Writes k and v [B, T, heads, D] (None: not) to the host cache; -> (q turned [B, T, Hq, D], its bound, live [B, T],
    bounds of the K planes)."""
    rot = cache.d if rot is None else rot
    some = next(x for x in (q, k, v) if x is not None)
    B, T = some.shape[:2]
    live = np.zeros((B, T), bool)
    out, bound = (np.zeros((B, T, 0 if q is None else q.shape[2], cache.d)) for _ in "ab")
    k_bound = np.zeros(cache.planes["k"].shape)
    for b in range(B):
        for t in range(T if counts is None else min(counts[b], T)):
            live[b, t] = True
            pos = positions[b] + t
            turn = lambda x: rotate(x[b, t].astype(np.float64), pos if angles is None else angles[b][t], base, rot, interleaved, divisors)
            if q is not None:
                out[b, t], bound[b, t] = turn(q)
            at = cache.at(b, pos)
            if at is None:
                continue
            if k is not None:
                y, off = turn(k)
                cache.write("k", b, pos, y, layer)
                if cache.dtype == 1:                     # rounded to fp16: half a step, and half of 2^-24 next to zero
                    off = off + np.abs(y) * 2.0 ** -11 + 2.0 ** -25
                k_bound[layer, at[0], :, at[1]] = off + np.abs(y) * 2.0 ** -24
            if v is not None:
                cache.write("v", b, pos, v[b, t], layer)
    return out, bound, live, k_bound


# ---- attention -----------------------------------------------------------------------

def attention(cache, q, lens, counts=None, parents=None, window=0, cap=0.0, scale=None, layer=0):
    """q [B, T, Hq, D] -> (out float64, bound, live [B, T]): rows that are not live are left alone.

    The bound: a score is off by at most A (2^-22 + (D + 16) 2^-24), A = scale sum |q||k|: the query's two fp16 parts
    keep 2^-22 of each element, and its products' sum is rounded at most D + 16 times (scaling, chains, the exponent's
    argument); a soft cap adds 4 roundings of a number up to 2 cap. Weights are off by that, by 2^-22 for the exponential
    and 2^-22 for two fp16 parts, which lose what is below 2^-36 of the largest weight (weights, at most 16, times 2^11, next to fp16's 2^-25); the sums over n keys by a
    rounding a key and 64 for their joining. An output is a weighted mean, so all of it is relative to the weighted
    mean of |v|, twice for the denominator."""
    B, T, Hq, D = q.shape
    scale = D ** -0.5 if scale is None else scale
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    live = np.zeros((B, T), bool)
    g = Hq // cache.heads
    for b in range(B):
        n = min(max(int(lens[b]), 0), cache.cap)
        cnt = T if counts is None else min(max(int(counts[b]), 0), T)
        live[b, :cnt] = True
        k, has = cache.rows_of("k", b, n, layer)
        v, _ = cache.rows_of("v", b, n, layer)
        base = n - cnt
        up = chain(T) if parents is None else parents[b]
        lines = [line(up, t) for t in range(cnt)]
        for t in range(cnt):
            pos = base + len(lines[t]) - 1
            keys = [(j, j) for j in range(max(base, 0))] + [(base + i, base + len(lines[i]) - 1) for i in lines[t] if base + i >= 0]
            see = np.zeros(n, bool)
            for j, at in keys:
                see[j] = has[j] and (window <= 0 or pos - at < window)
            if not see.any():
                continue
            for kv in range(cache.heads):
                kk, vv = k[kv][see], v[kv][see]
                x = q[b, t, kv * g:(kv + 1) * g].astype(np.float64)
                with np.errstate(all="ignore"):
                    s = x @ kk.T * scale
                    off = np.abs(x) @ np.abs(kk).T * scale * (2.0 ** -22 + (D + 16) * 2.0 ** -24)
                    if cap > 0:
                        s = cap * np.tanh(s / cap)
                        off = off + 2 * cap * 4 * 2.0 ** -24
                    off = np.where(np.isfinite(s), off, 0.0)            # a score that is not finite is exact, or its row is NaN
                    w = np.exp(s - s.max(-1, keepdims=True))
                    w = np.where((s == -np.inf).all(-1, keepdims=True), 0.0, w / w.sum(-1, keepdims=True))
                    out[b, t, kv * g:(kv + 1) * g] = w @ vv
                    size = np.abs(vv)
                    bound[b, t, kv * g:(kv + 1) * g] = (2 * (w @ size) * (off.max(-1, keepdims=True) + 2.0 ** -21 + (see.sum() + 64) * 2.0 ** -24)
                                                        + see.sum() * 2.0 ** -36 * size.max(initial=0.0, where=np.isfinite(size)))
    return out, bound, live


# ---- accepted rows -------------------------------------------------------------------

def accept(cache, lens, counts, parents, tokens, choices):
    """Moves the accepted rows of the host cache; -> new_lens, path, accepted, next."""
    B, T = tokens.shape
    new_lens, path, accepted, after = (np.zeros(B, np.int32), np.full((B, T), -1, np.int32), np.zeros(B, np.int32), np.full(B, -1, np.int32))
    for b in range(B):
        n = min(max(int(lens[b]), 0), cache.cap)
        cnt = T if counts is None else min(max(int(counts[b]), 0), T)
        up = chain(T) if parents is None else parents[b]
        walk = [0] if cnt else []
        while walk:
            on = [i for i in range(walk[-1] + 1, cnt) if up[i] == walk[-1] and tokens[b, i] == choices[b, walk[-1]]]
            if not on:
                break
            walk.append(on[0])
        path[b, :len(walk)], accepted[b], new_lens[b] = walk, len(walk), n - cnt + len(walk)
        if walk:
            after[b] = choices[b, walk[-1]]
        for i, r in enumerate(walk):
            src, dst = cache.at(b, n - cnt + r), cache.at(b, n - cnt + i)
            if src is not None and dst is not None:
                for w in "kv":
                    cache.planes[w][:, dst[0], :, dst[1]] = cache.planes[w][:, src[0], :, src[1]]
    return new_lens, path, accepted, after
