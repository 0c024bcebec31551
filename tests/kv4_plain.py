"""The 4-bit KV cache in plain numpy: its encoder and decoder bit by bit, and
attention over it in float64 with a bound on what fp32 work may be off by."""
from __future__ import annotations

import numpy as np


def encode(x):
    """[..., D] fp32/fp16 -> (codes uint8 [..., D/2], scales float16 [..., D/32])."""
    x = np.asarray(x, np.float32).astype(np.float64)
    b = x.reshape(*x.shape[:-1], -1, 32)
    bad = ~np.isfinite(b).all(-1)
    b = np.where(bad[..., None], 0.0, b)
    lo, hi = b.min(-1), b.max(-1)
    neg = -lo >= hi
    step = np.where(neg, -lo, hi) / 8
    # 8 significant bits: multiples of 2^(e - 7) for a step in [2^e, 2^(e+1)), of 2^-24 at the least; ties to even.
    e = np.frexp(step)[1] - 1
    quantum = np.ldexp(1.0, np.maximum(e - 7, -24))
    step = np.minimum(np.rint(step / quantum) * quantum, 8160.0)
    d = np.where(neg, step, -step)
    d = np.where(step == 0, 0.0, d)
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.clip(np.floor(b / d[..., None] + 0.5), -8, 7)
    q = np.where((step == 0)[..., None], 0, q)
    c = (q + 8).astype(np.uint8)
    scales = np.where(bad, np.nan, d).astype(np.float16)
    assert np.array_equal(scales.astype(np.float64)[~bad], d[~bad])
    c = np.where(bad[..., None], 8, c).astype(np.uint8)
    codes = c[..., :16] | (c[..., 16:] << 4)
    return codes.reshape(*x.shape[:-1], -1), scales


def decode(codes, scales):
    """Values as float16 numbers, (code - 8) * scale rounded once."""
    c = codes.reshape(*codes.shape[:-1], -1, 16)
    q = np.concatenate([c & 15, c >> 4], -1).astype(np.float16) - np.float16(8)
    with np.errstate(invalid="ignore", over="ignore"):
        return (q * scales[..., None]).reshape(*codes.shape[:-1], -1)


class Cache:
    """Host planes of one cache: contiguous (page = 0) or paged."""

    def __init__(self, seqs, heads, d, cap, page=0, seed=0, fill=0xAB):
        rng = np.random.default_rng(seed)
        self.seqs, self.heads, self.d, self.page = seqs, heads, d, page
        if page:
            self.per = -(-cap // page)
            self.s, self.rows = seqs * self.per + 2, page
            self.table = rng.permutation(self.s)[:seqs * self.per].reshape(seqs, self.per).astype(np.int32)
            self.cap = self.per * page
        else:
            self.per, self.s, self.rows, self.table, self.cap = 1, seqs, cap, None, cap
        # What nothing was written to holds garbage: here NaN scales.
        self.codes = {w: np.full((self.s, heads, self.rows, d // 2), fill, np.uint8) for w in "kv"}
        self.scales = {w: np.full((self.s, heads, d // 32, self.rows), np.nan, np.float16) for w in "kv"}

    def at(self, b, pos):
        """(plane, row) of a position, None where the cache has no such row."""
        if pos < 0 or pos >= self.cap:
            return None
        if self.table is None:
            return b, pos
        s = int(self.table[b, pos // self.page])
        return (s, pos % self.page) if 0 <= s < self.s else None

    def write(self, which, b, pos, x):
        """x [heads, D] at position pos of sequence b."""
        at = self.at(b, pos)
        if at is None:
            return
        codes, scales = encode(x)
        self.codes[which][at[0], :, at[1]] = codes
        self.scales[which][at[0], :, :, at[1]] = scales

    def fill(self, lens, seed=1):
        rng = np.random.default_rng(seed)
        for which in "kv":
            for b, n in enumerate(lens):
                x = rng.standard_normal((max(int(n), 0), self.heads, self.d)).astype(np.float32)
                if which == "k":
                    x *= np.exp(0.5 * np.random.default_rng(seed + 7).standard_normal((self.heads, self.d))).astype(np.float32)
                for pos in range(max(int(n), 0)):
                    self.write(which, b, pos, x[pos])

    def rows_of(self, which, b, n):
        """The values [heads, n, D] of the first n positions, and which of them the cache has."""
        out = np.zeros((self.heads, n, self.d), np.float16)
        has = np.zeros(n, bool)
        for pos in range(n):
            at = self.at(b, pos)
            if at is not None:
                has[pos] = True
                out[:, pos] = decode(self.codes[which][at[0], :, at[1]], self.scales[which][at[0], :, :, at[1]])
        return out, has


def attention(cache, q, lens, counts=None, causal=True, window=0, cap=0.0, scale=None):
    """q [B, T, Hq, D] -> (out float64, bound, live [B, T]): rows that are not live are left alone.

    The bound: a score is off by at most A (2^-22 + (D + 16) 2^-24), A = scale sum |q||k|: the query's two fp16 parts
    keep 2^-22 of each element, and its products' sum is rounded at most D + 16 times (scaling, chains, the exponent's
    argument); a soft cap adds 4 roundings of a number up to 2 cap. Weights are off by that, and by 2^-22 for their two
    parts and 2^-22 for the exponential; the sums over n keys by a rounding per 16 keys and 64 for their joining.
    An output is a weighted mean, so all of it is relative to the weighted mean of |v|, twice for the denominator."""
    B, T, Hq, D = q.shape
    scale = D ** -0.5 if scale is None else scale
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    live = np.zeros((B, T), bool)
    g = Hq // cache.heads
    for b in range(B):
        n = min(max(int(lens[b]), 0), cache.cap)
        cnt = T if counts is None else min(max(int(counts[b]), 0), T)
        live[b, :cnt] = True
        k, has = cache.rows_of("k", b, n)
        v, _ = cache.rows_of("v", b, n)
        k, v = k.astype(np.float64), v.astype(np.float64)
        j = np.arange(n)
        for t in range(cnt):
            pos = n - cnt + t
            see = has & (j <= pos if causal else True)
            if window > 0:
                see = see & (j > pos - window)
            if not see.any():
                continue
            for h in range(Hq):
                kk, vv = k[h // g][see], v[h // g][see]
                x = q[b, t, h].astype(np.float64)
                with np.errstate(all="ignore"):
                    s = kk @ x * scale
                    a = np.abs(kk) @ np.abs(x) * scale
                    off = a * (2.0 ** -22 + (D + 16) * 2.0 ** -24)
                    if cap > 0:
                        s = cap * np.tanh(s / cap)
                        off = off + 2 * cap * 4 * 2.0 ** -24
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    out[b, t, h] = w @ vv
                    mean = w @ np.abs(vv)
                    bound[b, t, h] = 2 * mean * (off.max() + 2.0 ** -21 + (see.sum() / 16 + 64) * 2.0 ** -24)
    return out, bound, live


def one_hot_keys(d, n=40, seed=0):
    """A cache whose keys are one number in [1, 2) and zeros: a score is one product, off by all of its query element's
    error, where the bound allows a sum of D of them. Queries for it: one_hot_query."""
    rng = np.random.default_rng(seed)
    host = Cache(1, 1, d, -(-n // 16) * 16)
    for pos in range(n):
        k = np.zeros((1, d), np.float32)
        k[0, rng.integers(0, d)] = rng.choice([-1.0, 1.0]) * rng.uniform(1, 2)
        host.write("k", 0, pos, k)
        host.write("v", 0, pos, rng.standard_normal((1, d)).astype(np.float32))
    return host


def one_hot_query(d, t, g):
    rng = np.random.default_rng(d + t)
    return (rng.uniform(1, 2, (1, t, g, d)) * rng.choice([-1, 1], (1, t, g, d))).astype(np.float32)


def in_fp16_parts(cache, q, n, scale, query_parts, weight_parts):
    """Causal attention of one sequence and KV head with queries and weights in one or two fp16 parts, else in float64."""
    k, v = (cache.rows_of(w, 0, n)[0][0].astype(np.float64) for w in "kv")

    def parts(x, count):
        first = x.astype(np.float16).astype(np.float64)
        return first if count == 1 else first + (x - first).astype(np.float16).astype(np.float64)

    out = np.zeros(q.shape)
    for t in range(q.shape[1]):
        seen = n - q.shape[1] + t + 1
        for h in range(q.shape[2]):
            x = q[0, t, h].astype(np.float64) * scale / np.log(2.0)
            e = int(np.frexp(np.abs(x).max())[1])
            s = k[:seen] @ parts(np.ldexp(x, 15 - e), query_parts) * 2.0 ** (e - 15)
            w = parts(np.exp2(s - s.max()) * 8192, weight_parts)
            out[0, t, h] = w @ v[:seen] / w.sum()
    return out
