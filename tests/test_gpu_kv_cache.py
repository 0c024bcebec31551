"""fp16 and fp32 KV caches on the GPU: rows rotated and appended, attention of
trees and chains of drafted rows against float64 within the bounds that
``kv_plain`` derives, accepted rows bit for bit, and the three together."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import kv_plain as plain
from conftest import fresh_thread, scratch_held

pytestmark = pytest.mark.gpu

F32, F16 = 0, 1
ROOM = 1 << 28                                              # of a large cache, see Device
POISON = -77.0


class Device:
    """A host cache's planes on the GPU and the description the calls take. room: bytes that one layer's rows are to take at
    the least, in which the host's are the first; attention shares its work out by what a cache has room for."""

    def __init__(self, rocm, host, room=0):
        put = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
        self.host = host
        self.planes = {w: put(host.planes[w]) for w in "kv"}
        self.table = None if host.table is None else put(host.table)
        rows, per, cap = host.rows, host.per, -(-room // (2 * host.seqs * host.heads * host.d * host.planes["k"].itemsize))
        if host.page and cap > host.cap:                    # a wider table, without blocks past the host's
            per = -(-cap // host.page)
            table = torch.full((host.seqs, per), -1, dtype=torch.int32, device="cuda")
            table[:, :host.per] = self.table
            self.table = table
        elif cap > host.cap:
            rows = cap
            for w, x in self.planes.items():
                self.planes[w] = torch.full((*x.shape[:3], rows, x.shape[4]), float("nan"), dtype=x.dtype, device="cuda")
                self.planes[w][:, :, :, :host.rows] = x
        self.desc = rocm.KvCache(self.planes["k"].data_ptr(), self.planes["v"].data_ptr(), ptr(self.table), host.dtype, host.layers,
                                 host.seqs, host.heads, host.d, rows, host.s if host.page else 0, per if host.page else 0)
        torch.cuda.synchronize()

    def ref(self):
        return ctypes.byref(self.desc)

    def plane(self, w):
        torch.cuda.synchronize()
        return self.planes[w].cpu().numpy()


def ints(x):
    return None if x is None else torch.tensor(np.asarray(x), dtype=torch.int32).cuda()


def ptr(t):
    return None if t is None else t.data_ptr()


def attend(rocm, dev, q, lens, counts=None, parents=None, window=0, cap=0.0, scale=0.0, workspace=None, layer=0):
    B, T, Hq, _ = q.shape
    qd, ld, cd, pd = torch.from_numpy(q).cuda(), ints(lens), ints(counts), ints(parents)
    out = torch.full(q.shape, POISON, device="cuda")
    torch.cuda.synchronize()
    rocm.call("aljabr_rocm_kv_tree_attention", out.data_ptr(), qd.data_ptr(), dev.ref(), layer, ld.data_ptr(), ptr(cd), ptr(pd), T, Hq,
              scale, window, cap, ptr(workspace), 0 if workspace is None else workspace.numel())
    torch.cuda.synchronize()
    return out.cpu().numpy()


def check(got, want, bound, live):
    assert (got[~live] == POISON).all(), "rows behind a sequence's last were written"
    err = np.abs(got.astype(np.float64) - want)[live]
    assert (err <= bound[live] + 1e-30).all(), (np.nanmax(err), np.nanmax(err / (bound[live] + 1e-30)), np.isnan(err).sum())


def normal(seed, *shape):
    return np.random.default_rng(seed).standard_normal(shape).astype(np.float32)


# ---- appended rows ------------------------------------------------------------------

def lay_out(x, layout):
    """A float array [B, T, H, D] as (buffer, offset in elements, strides)."""
    b, t, h, d = x.shape
    if layout == "dense":
        return x.copy(), 0, (0, 0, 0)
    if layout == "heads":
        return np.ascontiguousarray(x.transpose(0, 2, 1, 3)), 0, (h * t * d, d, t * d)
    pad = 5 if layout == "odd" else 8                       # odd: rows off the wide loads' alignment
    row, off = h * d + pad, 4 if layout == "odd" else 4
    out = np.full((b, t, row), 9.0, x.dtype)
    out[:, :, off:][:, :, :h * d] = x.reshape(b, t, -1)
    return out, off, (t * row, row, d)


def append(rocm, dev, q, k, v, positions, counts=None, angles=None, base=1e4, rot=0, interleaved=0, divisors=None, layer=0,
           layouts=("dense", "dense"), turned=True):
    """Calls kv_append; -> q_out."""
    some = next(x for x in (q, k, v) if x is not None)
    b, t, dtype = some.shape[0], some.shape[1], F16 if some.dtype == np.float16 else F32
    bufs = [None if x is None else lay_out(x, lay) for x, lay in ((q, layouts[0]), (k, layouts[1]), (v, layouts[1]))]
    devs = [None if x is None else torch.from_numpy(x[0]).cuda() for x in bufs]
    ptrs = [None if x is None else y.data_ptr() + x[1] * some.itemsize for x, y in zip(bufs, devs)]
    hq = 0 if q is None else q.shape[2]
    out = torch.full((b, t, max(hq, 1), dev.host.d), POISON, device="cuda")
    pos, cnt, ang = ints(positions), ints(counts), ints(angles)
    div = None if divisors is None else torch.from_numpy(divisors).cuda()
    rotation = rocm.Rotation(base, rot, interleaved, ptr(div))
    torch.cuda.synchronize()
    rocm.call("aljabr_rocm_kv_append", dev.ref(), layer, None if q is None else out.data_ptr(), *ptrs, pos.data_ptr(), ptr(cnt), ptr(ang),
              t, hq, *((0, 0, 0) if q is None else bufs[0][2]), *((0, 0, 0) if k is None and v is None else (bufs[1] or bufs[2])[2]), dtype,
              ctypes.byref(rotation) if turned else None)
    torch.cuda.synchronize()
    return out.cpu().numpy()


def check_planes(dev, k_bound=None):
    """The planes on the GPU are the host's: K within a bound, V and what nothing wrote bit for bit."""
    assert np.array_equal(dev.plane("v"), dev.host.planes["v"], equal_nan=True)
    got, want = dev.plane("k"), dev.host.planes["k"]
    if k_bound is None:
        assert np.array_equal(got, want, equal_nan=True)
        return
    loose = k_bound > 0
    assert np.array_equal(got[~loose], want[~loose], equal_nan=True)
    with np.errstate(invalid="ignore"):
        err = np.abs(got.astype(np.float64) - want.astype(np.float64))
    # The host's own rounding to the cache's type is within the bound's terms for it once more.
    assert (err[loose] <= 2 * k_bound[loose]).all(), (err[loose] / k_bound[loose]).max()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("t,page,src,layouts,rot,interleaved,hkv,g", [
    (1, 0, np.float32, ("dense", "dense"), 0, 0, 2, 4), (1, 16, np.float16, ("heads", "row"), 32, 1, 1, 1),
    (5, 48, np.float32, ("row", "odd"), 56, 0, 3, 2), (7, 0, np.float16, ("odd", "odd"), 8, 1, 2, 3),
    (16, 32, np.float32, ("row", "row"), 0, 1, 2, 8), (37, 16, np.float32, ("heads", "heads"), 24, 0, 1, 7),
    (70, 0, np.float16, ("dense", "heads"), 0, 0, 2, 2), (33, 64, np.float16, ("row", "dense"), 64, 1, 3, 1)])
def test_append(rocm, d, dtype, t, page, src, layouts, rot, interleaved, hkv, g):
    b = 3
    q, k, v = (normal(s + d, b, t, n, d).astype(src) for s, n in ((1, hkv * g), (2, hkv), (3, hkv)))
    host = plain.Cache(b, hkv, d, 97, page, dtype, layers=2)
    dev = Device(rocm, host)
    start, counts = [0, 11, 96 - t], [t, max(t - 2, 0), t]
    angles = np.random.default_rng(t).integers(0, 200000, (b, t)) if t % 2 else None
    divisors = np.random.default_rng(d).uniform(0.5, 40, d // 2).astype(np.float32) if page else None
    if divisors is not None:
        divisors[1], divisors[3] = 0.0, -2.0                # not positive: no division
    args = (q, k, v, start, counts, angles, 5e5)
    got = append(rocm, dev, *args, rot, interleaved, divisors, 1, layouts)
    want, bound, live, k_bound = plain.append(host, *args, rot or d, bool(interleaved), divisors, 1)
    check(got, want, bound + np.abs(want) * 2.0 ** -24, live)
    check_planes(dev, k_bound)


@pytest.mark.parametrize("dtype", [F32, F16])
def test_append_without_rotation_copies(rocm, dtype):
    host = plain.Cache(2, 2, 128, 40, 0, dtype)
    dev = Device(rocm, host)
    q, k, v = normal(1, 2, 6, 4, 128), normal(2, 2, 6, 2, 128), normal(3, 2, 6, 2, 128)
    k[0, 0, 0, :4] = [np.inf, -np.inf, np.nan, 1e6]         # 1e6 is past fp16: an infinity there
    got = append(rocm, dev, q, k, v, [0, 34], turned=False)
    assert np.array_equal(got, q)
    plain.append(host, None, k, v, [0, 34], rot=0)
    check_planes(dev)


def test_append_of_each_alone(rocm):
    host = plain.Cache(1, 2, 64, 32)
    dev = Device(rocm, host)
    q, k, v = (normal(s, 1, 3, 2, 64) for s in (1, 2, 3))
    append(rocm, dev, None, None, v, [2])
    plain.append(host, None, None, v, [2])
    check_planes(dev)
    got = append(rocm, dev, q, None, None, [5])
    want, bound, live, _ = plain.append(host, q, None, None, [5])
    check(got, want, bound + np.abs(want) * 2.0 ** -24, live)
    check_planes(dev)
    append(rocm, dev, None, k, None, [2])
    _, _, _, k_bound = plain.append(host, None, k, None, [2])
    check_planes(dev, k_bound)


def test_append_in_place(rocm):
    """q_out is Q."""
    host = plain.Cache(2, 1, 128, 32)
    dev = Device(rocm, host)
    q, k = normal(1, 2, 4, 4, 128), normal(2, 2, 4, 1, 128)
    qd, kd, pos, cnt = torch.from_numpy(q).cuda(), torch.from_numpy(k).cuda(), ints([3, 9]), ints([4, 2])
    rotation = rocm.Rotation(1e4, 0, 0, None)
    torch.cuda.synchronize()
    rocm.call("aljabr_rocm_kv_append", dev.ref(), 0, qd.data_ptr(), qd.data_ptr(), kd.data_ptr(), kd.data_ptr(), pos.data_ptr(),
              cnt.data_ptr(), None, 4, 4, 0, 0, 0, 0, 0, 0, F32, ctypes.byref(rotation))
    got = qd.cpu().numpy()
    want, bound, live, k_bound = plain.append(host, q, k, k, [3, 9], [4, 2])
    assert np.array_equal(got[~live], q[~live])
    assert (np.abs(got - want)[live] <= (bound + np.abs(want) * 2.0 ** -24)[live]).all()
    check_planes(dev, k_bound)


def test_append_of_rows_the_cache_does_not_have(rocm):
    b, t = 5, 8
    host = plain.Cache(b, 2, 64, 48, 16)
    host.table[0, 1], host.table[1, 0], host.table[2, 2] = -1, host.s, 2 ** 31 - 1
    dev = Device(rocm, host)
    q, k, v = normal(1, b, t, 4, 64), normal(2, b, t, 2, 64), normal(3, b, t, 2, 64)
    start, counts = [12, 12, -3, 44, 2 ** 31 - 4], [t, t, t, t, 2 ** 31 - 1]
    args = (q, k, v, start, counts, np.zeros((b, t), int) + 7)
    got = append(rocm, dev, *args)
    want, bound, live, k_bound = plain.append(host, *args)
    check(got, want, bound + np.abs(want) * 2.0 ** -24, live)          # the queries of dropped rows are turned all the same
    check_planes(dev, k_bound)


@pytest.mark.parametrize("at", [0, 1, 131071, 2 ** 24 + 1, 2 ** 30 - 1, 2 ** 31 - 1, -5, -2 ** 31])
@pytest.mark.parametrize("base", [1e4, 5e5, 1.0, 0.5, 1e30])
def test_far_positions(rocm, at, base):
    host = plain.Cache(1, 1, 128, 16, 0, F32)
    dev = Device(rocm, host)
    q = normal(1, 1, 1, 2, 128)
    got = append(rocm, dev, q, None, None, [0], None, [[at]], base)
    want, bound, live, _ = plain.append(host, q, None, None, [0], None, [[at]], base)
    check(got, want, bound + np.abs(want) * 2.0 ** -24, live)


def test_near_positions_turn_as_rope_does(rocm):
    """aljabr_rocm_rope of the same rows: its angles, rounded to fp32, are off by 2^-23 of themselves."""
    host = plain.Cache(1, 1, 128, 64, 0, F32)
    dev = Device(rocm, host)
    x = normal(1, 1, 50, 4, 128)
    got = append(rocm, dev, x, None, None, [0])
    xd, pos = torch.from_numpy(x).cuda(), ints(np.arange(50))
    torch.cuda.synchronize()
    rocm.call("aljabr_rocm_rope", xd.data_ptr(), pos.data_ptr(), 50, 4, 128, 1e4)
    pair = np.abs(x[..., :64]) + np.abs(x[..., 64:])
    assert (np.abs(got - xd.cpu().numpy()) <= np.concatenate([pair, pair], -1) * (50 * 2.0 ** -23 + 12 * 2.0 ** -24)).all()


@pytest.mark.parametrize("paged", [0, 1])
def test_planes_past_32_bits(rocm, paged):
    """Rows at the end of planes of 8 GiB, written and seen through a window; the second of two layers."""
    h, d, n, seen, t, g = 2, 256, 1 << 22, 80, 5, 4
    rows, blocks = (16, n // 16) if paged else (n, 1)
    small = plain.Cache(1, h, d, 96)                                   # the last rows alone
    planes = {w: torch.empty(2 * blocks * h * rows * d, dtype=torch.float16, device="cuda") for w in "kv"}
    table = torch.arange(n // 16, dtype=torch.int32, device="cuda") if paged else None
    desc = rocm.KvCache(planes["k"].data_ptr(), planes["v"].data_ptr(), ptr(table), F16, 2, 1, h, d, rows, blocks if paged else 0,
                        n // 16 if paged else 0)
    need = ctypes.c_size_t()
    rocm.call("aljabr_rocm_kv_cache_bytes", ctypes.byref(desc), ctypes.byref(need))
    assert need.value == 2 * planes["k"].numel()
    x = normal(t, 2, 1, seen, h, d)
    plain.append(small, None, x[0], x[1], [0], rot=0)
    xd, pos, lens = torch.from_numpy(x).cuda(), ints([n - seen]), ints([n])
    torch.cuda.synchronize()
    rocm.call("aljabr_rocm_kv_append", ctypes.byref(desc), 1, None, None, xd[0].data_ptr(), xd[1].data_ptr(), pos.data_ptr(), None, None,
              seen, 0, 0, 0, 0, 0, 0, 0, F32, None)
    parents = plain.random_parents(np.random.default_rng(0), 1, t)
    q = normal(2, 1, t, h * g, d)
    qd, pd, out = torch.from_numpy(q).cuda(), ints(parents), torch.full(q.shape, POISON, device="cuda")
    torch.cuda.synchronize()
    rocm.call("aljabr_rocm_kv_tree_attention", out.data_ptr(), qd.data_ptr(), ctypes.byref(desc), 1, lens.data_ptr(), None, pd.data_ptr(),
              t, h * g, 0.0, 64, 0.0, None, 0)
    check(out.cpu().numpy(), *plain.attention(small, q, [seen], None, parents, window=64))
    tokens = np.arange(t)[None]
    choices = np.full((1, t), -1)
    last = plain.line(parents[0], t - 1)[::-1]
    for a, b in zip(last, last[1:]):
        choices[0, a] = tokens[0, b]
    outs = [torch.zeros(t, dtype=torch.int32, device="cuda") for _ in range(4)]
    tk, ch = ints(tokens), ints(choices)
    torch.cuda.synchronize()
    rocm.call("aljabr_rocm_kv_tree_accept", ctypes.byref(desc), *[o.data_ptr() for o in outs], lens.data_ptr(), None, pd.data_ptr(),
              tk.data_ptr(), ch.data_ptr(), t)
    want = plain.accept(small, [seen], None, parents, tokens, choices)
    assert outs[1].cpu().tolist() == want[1][0].tolist() and len(last) > 1
    tail = planes["v"].view(2, blocks, h, rows, d)[1]
    tail = tail[0, :, -16:] if not paged else tail[-1]
    assert np.array_equal(tail.cpu().numpy(), small.planes["v"][0, 0, :, 64:80])


# ---- attention ---------------------------------------------------------------------

SHAPES = [(1, 1), (8, 4), (4, 8), (2, 3), (1, 16), (3, 7)]           # (KV heads, query heads of each)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("hkv,g", SHAPES)
@pytest.mark.parametrize("page", [0, 16, 48])
def test_decode(rocm, d, dtype, hkv, g, page):
    lens = [1, 33, 200, 0]
    host = plain.Cache(4, hkv, d, 203, page, dtype)
    host.fill(lens)
    q = normal(d + g, 4, 1, hkv * g, d)
    got = attend(rocm, Device(rocm, host), q, lens, [1, 1, 1, 0] if g == 3 else None)
    check(got, *plain.attention(host, q, lens, [1, 1, 1, 0] if g == 3 else None))
    assert g == 3 or not got[3].any()                                 # no key: zeros


@pytest.mark.parametrize("room", [0, ROOM])
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 127, 128, 129, 255, 257, 511, 1000, 2047])
def test_lengths(rocm, room, n, dtype):
    host = plain.Cache(1, 2, 128, 2047, 0, dtype)
    host.fill([n], seed=n)
    q = normal(n, 1, 1, 8, 128)
    check(attend(rocm, Device(rocm, host, room), q, [n]), *plain.attention(host, q, [n]))


@pytest.mark.parametrize("room", [0, ROOM])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("t,hkv,g", [(2, 2, 4), (5, 2, 2), (8, 1, 8), (9, 2, 1), (17, 2, 4), (26, 2, 1), (40, 1, 3), (70, 2, 2)])
@pytest.mark.parametrize("window,cap", [(0, 0.0), (20, 0.0), (40, 5.0), (1, 0.0), (-3, 0.0), (2 ** 31 - 1, 0.0)])
@pytest.mark.parametrize("tree", [0, 1, 2])
def test_several_rows(rocm, room, d, dtype, t, hkv, g, window, cap, tree):
    lens, counts = [t, 100, 3, 150], [t, max(t - 3, 1), t, 0]         # the third: more rows than keys
    host = plain.Cache(4, hkv, d, 157, 16 if t % 2 else 0, dtype)
    host.fill(lens)
    parents = plain.random_parents(np.random.default_rng(t), 4, t, deep=tree == 2) if tree else None
    q = normal(t, 4, t, hkv * g, d)
    got = attend(rocm, Device(rocm, host, room), q, lens, counts, parents, window, cap)
    check(got, *plain.attention(host, q, lens, counts, parents, window, cap))


@pytest.mark.parametrize("room", [0, ROOM])
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("t", [31, 32, 33, 64, 65, 128, 200, 255, 256])
@pytest.mark.parametrize("shape", ["chain", "deep", "star", "forest", "wild"])
@pytest.mark.parametrize("window", [0, 5, 33])
def test_trees_of_every_size(rocm, room, t, shape, window, dtype):
    rng = np.random.default_rng(t)
    b = 2
    if shape == "wild":                                               # numbers that are no earlier rows stand for none
        parents = rng.integers(-5, t + 5, (b, t)).astype(np.int32)
        parents[0, 0], parents[1, 0], parents[0, t - 1] = 2 ** 31 - 1, 3, -2 ** 31
    elif shape == "forest":
        parents = np.where(rng.random((b, t)) < 0.3, -1, plain.random_parents(rng, b, t)).astype(np.int32)
    else:
        parents = {"chain": np.stack([plain.chain(t)] * b), "deep": plain.random_parents(rng, b, t, True),
                   "star": np.where(np.arange(t) == 0, -1, 0)[None].repeat(b, 0).astype(np.int32)}[shape]
    lens, counts = [t + 45, t + 3], [t, t - 1]
    host = plain.Cache(b, 1, 64, t + 50, 16 if t % 2 else 0, dtype)
    host.fill(lens)
    q = normal(t, b, t, 2, 64)
    got = attend(rocm, Device(rocm, host, room), q, lens, counts, parents, window)
    check(got, *plain.attention(host, q, lens, counts, parents, window))


@pytest.mark.parametrize("room", [0, ROOM])
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("t", [1, 5, 20])
def test_scale_and_large_scores(rocm, room, dtype, t):
    host = plain.Cache(1, 2, 128, 304, 0, dtype)
    host.fill([300])
    dev = Device(rocm, host, room)
    for scale, size in ((0.5, 1.0), (2.0, 30.0), (1e-3, 1e-20), (1e-4, 1e6)):
        q = normal(3, 1, t, 8, 128) * np.float32(size)
        check(attend(rocm, dev, q, [300], scale=scale), *plain.attention(host, q, [300], scale=scale))


@pytest.mark.parametrize("room", [0, ROOM])
def test_fp32_values_of_any_size(rocm, room):
    """What fp16 does not hold: keys of 1e-9 against queries of 1e9, values from 1e-30 to 1e30."""
    host = plain.Cache(1, 2, 128, 90, 0, F32)
    host.fill([90])
    host.planes["k"] *= np.float32(1e-9)
    host.planes["v"] *= np.exp(np.random.default_rng(4).uniform(-60, 60, 128)).astype(np.float32)
    for t in (1, 20):
        q = normal(t, 1, t, 8, 128) * np.float32(1e9)
        check(attend(rocm, Device(rocm, host, room), q, [90]), *plain.attention(host, q, [90]))


@pytest.mark.parametrize("room", [0, ROOM])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("t", [1, 6, 12, 40])
def test_bad_blocks_hold_no_keys(rocm, room, d, dtype, t):
    lens = [90, 90, 90, 20]
    host = plain.Cache(4, 2, d, 96, 16, dtype)
    host.fill(lens)
    host.table[0, 2], host.table[1, 0], host.table[1, 5], host.table[3, :] = -1, host.s, 2 ** 31 - 1, -5
    parents = plain.random_parents(np.random.default_rng(0), 4, t) if t in (6, 12) else None
    q = normal(6, 4, t, 8, d)
    got = attend(rocm, Device(rocm, host, room), q, lens, None, parents)
    check(got, *plain.attention(host, q, lens, None, parents))
    assert not got[3].any()


def test_lengths_past_the_cache_are_clamped(rocm):
    host = plain.Cache(2, 2, 64, 37)
    host.fill([37, 37])
    q = normal(7, 2, 1, 4, 64)
    got = attend(rocm, Device(rocm, host), q, [2 ** 31 - 1, -7])
    check(got, *plain.attention(host, q, [37, 0]))


@pytest.mark.parametrize("room", [0, ROOM])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("t,tree", [(4, 0), (12, 0), (40, 0), (4, 1), (12, 1), (40, 1)])
def test_values_that_are_not_finite_reach_only_rows_that_see_them(rocm, room, value, which, d, dtype, t, tree):
    """One element of one drafted row's key or value in one head: rows outside its line are as without it, and the others
    as float64 has them (an infinite score takes its row to NaN, or is a weight of zero)."""
    n = 100
    host = plain.Cache(1, 2, d, 128, 0, dtype)
    host.fill([n])
    parents = plain.random_parents(np.random.default_rng(t), 1, t) if tree else None
    q = normal(8, 1, t, 8, d)
    for row in (1, t - 2):
        saved = host.planes[which].copy()
        x = host.planes[which][0, 0, :, n - t + row].copy()
        x[1, 37] = value
        host.write(which, 0, n - t + row, x)
        want, bound, live = plain.attention(host, q, [n], None, parents)
        got = attend(rocm, Device(rocm, host, room), q, [n], None, parents)
        fine = np.isfinite(want)
        assert not fine.all() or which == "k"
        assert np.array_equal(got[~fine], want[~fine].astype(np.float32), equal_nan=True)
        assert (np.abs(got[fine] - want[fine]) <= bound[fine]).all()
        host.planes[which] = saved


@pytest.mark.parametrize("value", [np.nan, np.inf])
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("t", [1, 3, 40])
def test_window_leaves_values_behind_that_are_not_finite(rocm, value, dtype, d, t):
    """Cached keys before every window, and past the end, and one that only the first row still sees."""
    n, window = 150, 48
    host = plain.Cache(1, 1, d, 160, 16, dtype)
    host.fill([n])
    q = normal(9, 1, t, 4, d)
    first = n - t - window + 1                                         # of the first row's keys
    for pos in [*range(first), *range(n, 160)]:
        for w in "kv":
            host.write(w, 0, pos, np.full((1, d), value))
    clean = plain.attention(host, q, [n], window=window)
    assert np.isfinite(clean[0]).all()
    check(attend(rocm, Device(rocm, host), q, [n], window=window), *clean)
    host.write("v", 0, first, np.full((1, d), value))
    got = attend(rocm, Device(rocm, host), q, [n], window=window)
    want = plain.attention(host, q, [n], window=window)
    assert (got[0, 0] == np.float32(value)).all() or np.isnan(got[0, 0]).all()
    check(got[:, 1:], want[0][:, 1:], want[1][:, 1:], np.ones((1, t - 1), bool))


@pytest.mark.parametrize("room", [0, ROOM])
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("t", [1, 10, 40])
def test_infinite_scores(rocm, room, dtype, t):
    """Keys whose score is -inf weigh nothing, rows of such keys alone are zeros; +inf makes NaN."""
    host = plain.Cache(1, 1, 64, 64, 0, dtype)
    host.fill([50])
    host.planes["k"][0, 0, 0, :, 5] = 0
    host.planes["k"][0, 0, 0, 3, 5] = np.inf
    q = normal(1, 1, t, 4, 64)
    q[..., 5] = -np.abs(q[..., 5])
    want = plain.attention(host, q, [50])
    assert np.isfinite(want[0]).all()
    check(attend(rocm, Device(rocm, host, room), q, [50]), *want)
    assert np.isnan(attend(rocm, Device(rocm, host, room), -q, [50])).all()
    host.planes["k"][0, 0, 0, :, 5] = np.inf
    assert not attend(rocm, Device(rocm, host, room), q, [50]).any()


@pytest.mark.parametrize("room", [0, ROOM])
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("t", [1, 20, 50])
def test_workspace_of_any_size(rocm, room, dtype, t):
    host = plain.Cache(2, 2, 128, 1024, 32, dtype)
    lens = [1000, 700]
    host.fill(lens)
    dev = Device(rocm, host, room)
    q = normal(10, 2, t, 8, 128)
    want = plain.attention(host, q, lens)
    n = ctypes.c_size_t()
    rocm.call("aljabr_rocm_kv_tree_attention_workspace", dev.ref(), t, 8, ctypes.byref(n))
    assert n.value > 0
    for size in (n.value, n.value // 2, n.value // 3, 1000, 16, 0):
        ws = torch.full((max(size, 16) + 4096,), 0xCD, dtype=torch.uint8, device="cuda")
        got = attend(rocm, dev, q, lens, workspace=ws[:size] if size else None)
        check(got, *want)
        assert (ws[size:] == 0xCD).all()


@pytest.mark.parametrize("room", [0, ROOM])
@pytest.mark.parametrize("t,g", [(1, 4), (3, 8), (20, 4)])
@pytest.mark.parametrize("b,page", [(65, 0), (130, 16)])
@pytest.mark.parametrize("tree", [0, 1])
def test_many_uneven_sequences(rocm, room, b, page, t, g, tree):
    """More sequences than a wave has lanes, from no key to all of them, a few of them long."""
    rng = np.random.default_rng(b + t)
    lens = rng.integers(0, 200, b)
    lens[3], lens[64], lens[b - 1] = 1500, 900, 1
    counts = rng.integers(0, t + 1, b)
    host = plain.Cache(b, 1, 64, 1500, page, F16)
    host.fill(lens)
    parents = plain.random_parents(rng, b, t) if tree else None
    q = normal(b, b, t, g, 64)
    got = attend(rocm, Device(rocm, host, room), q, lens, counts, parents)
    check(got, *plain.attention(host, q, lens, counts, parents))


@pytest.mark.parametrize("b", [255, 256, 257, 320, 513, 900])
@pytest.mark.parametrize("t,g", [(1, 4), (6, 8)])
def test_hundreds_of_sequences(rocm, b, t, g):
    """Lengths are looked through 256 at once: the long sequences are in the first, the last and at the edges between."""
    rng = np.random.default_rng(b)
    lens, counts = rng.integers(0, 60, b), rng.integers(0, t + 1, b)
    for i in (0, 63, 64, 255, 256, 511, 512, b - 1):
        if i < b:
            lens[i], counts[i] = 300 + i % 7, t
    host = plain.Cache(b, 1, 64, 320, 16, F16)
    host.fill(lens)
    q = normal(b, b, t, g, 64)
    parents = plain.random_parents(rng, b, t)
    check(attend(rocm, Device(rocm, host), q, lens, counts, parents), *plain.attention(host, q, lens, counts, parents))


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("b,hkv", [(67, 1), (23, 3), (66, 1), (13, 5)])
@pytest.mark.parametrize("t,g", [(1, 4), (11, 7)])
def test_short_sequences_that_are_not_eights(rocm, b, hkv, dtype, t, g):
    """Caches of one chunk a sequence, whose KV heads and sequences are no multiple of the 8 XCDs."""
    rng = np.random.default_rng(b)
    lens, counts = rng.integers(t, 101, b), rng.integers(0, t + 1, b)
    host = plain.Cache(b, hkv, 64, 100, 0, dtype)
    host.fill(lens)
    q = normal(b, b, t, hkv * g, 64)
    check(attend(rocm, Device(rocm, host), q, lens, counts), *plain.attention(host, q, lens, counts))


def test_as_many_sequences_as_a_call_takes(rocm):
    """65535 sequences of up to 3 keys of one block, the last of 250: each row is a mean of values, or one of them."""
    b, d = 65535, 64
    host = plain.Cache(1, 1, d, 256, 16)
    host.fill([256])
    one = Device(rocm, host)
    table = one.table.expand(b, 16).contiguous()
    desc = rocm.KvCache.from_buffer_copy(one.desc)
    desc.sequences, desc.block_table = b, table.data_ptr()
    lens = np.arange(b) % 3
    lens[-1] = 250
    q = normal(1, 1, 1, 2, d)
    want = [plain.attention(host, q, [n]) for n in (0, 1, 2, 250)]
    qd, ld = torch.from_numpy(q).cuda().expand(b, 1, 2, d).contiguous(), ints(lens)
    out = torch.full((b, 1, 2, d), POISON, device="cuda")
    torch.cuda.synchronize()
    rocm.call("aljabr_rocm_kv_tree_attention", out.data_ptr(), qd.data_ptr(), ctypes.byref(desc), 0, ld.data_ptr(), None, None, 1, 2, 0.0, 0,
              0.0, None, 0)
    got = out.cpu().numpy()
    for i in range(3):
        err = np.abs(got[:-1][lens[:-1] == i] - want[i][0])
        assert (err <= want[i][1] + 1e-30).all()
    assert (np.abs(got[-1:] - want[3][0]) <= want[3][1]).all()


@pytest.mark.parametrize("room", [0, ROOM])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("g", [17, 33, 64, 130])
def test_one_token_of_many_heads(rocm, room, d, g):
    lens = [500, 31, 0]
    host = plain.Cache(3, 1, d, 512)
    host.fill(lens)
    q = normal(g, 3, 1, g, d)
    check(attend(rocm, Device(rocm, host, room), q, lens), *plain.attention(host, q, lens))


@pytest.mark.parametrize("room", [0, ROOM])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("t,ctx", [(300, 300), (130, 777)])
def test_chunks_of_prompts(rocm, room, d, dtype, t, ctx):
    host = plain.Cache(2, 2, d, ctx, 16, dtype)
    lens, counts = [ctx, ctx - 9], [t, t - 61]
    host.fill(lens)
    q = normal(t, 2, t, 8, d)
    for window in (0, 100):
        check(attend(rocm, Device(rocm, host, room), q, lens, counts, window=window), *plain.attention(host, q, lens, counts, window=window))


@pytest.mark.parametrize("d,dtype", [(64, F16), (128, F16), (256, F16), (128, F32)])
@pytest.mark.parametrize("t,b,g,tree", [(520, 2, 8, 0), (256, 4, 16, 1)])
def test_windows_of_many_rows(rocm, d, dtype, t, b, g, tree):
    """Windows that end inside the cached keys, and inside the rows' own, of thousands of rows a KV head."""
    lens, counts = [1300, 777, 650, 500][:b], [t, t - 71, t, t - 5][:b]
    host = plain.Cache(b, 2, d, 1310, 16 if tree else 0, dtype)
    host.fill(lens)
    parents = plain.random_parents(np.random.default_rng(t), b, t, deep=True) if tree else None
    q = normal(t, b, t, 2 * g, d)
    for window in (610, 130):
        got = attend(rocm, Device(rocm, host, ROOM), q, lens, counts, parents, window)
        check(got, *plain.attention(host, q, lens, counts, parents, window))


@pytest.mark.parametrize("page", [0, 16])
@pytest.mark.parametrize("d,t,g", [(128, 1, 4), (64, 6, 4), (256, 12, 4), (64, 40, 4), (128, 64, 4)])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_replayed_with_other_lengths(rocm, page, d, t, g, dtype):
    """A captured call reads lengths, counts and parents of its replay, and gives an eager call's bits."""
    b, hkv = 3, 2
    host = plain.Cache(b, hkv, d, 904, page, dtype)
    host.fill([900] * b)
    dev, q = Device(rocm, host, ROOM), normal(t, b, t, hkv * g, d)
    need = ctypes.c_size_t()
    rocm.call("aljabr_rocm_kv_tree_attention_workspace", dev.ref(), t, hkv * g, ctypes.byref(need))
    ws = [torch.empty(max(need.value, 16), dtype=torch.uint8, device="cuda") for _ in range(2)]
    rng = np.random.default_rng(t)
    runs = [([900, 40 + t, 333], [t, max(t - 2, 1), t]), ([t, 0, 900], [t, 0, 0]), ([t + 1, 899, 700], [1, t, t])]
    trees = [plain.random_parents(rng, b, t) for _ in runs]
    eager = [attend(rocm, dev, q, lens, counts, up, workspace=ws[0]) for (lens, counts), up in zip(runs, trees)]
    for got, (lens, counts), up in zip(eager, runs, trees):
        check(got, *plain.attention(host, q, lens, counts, up))
    qd, out = torch.from_numpy(q).cuda(), torch.empty(q.shape, device="cuda")
    lens, counts, up = (torch.zeros(s, dtype=torch.int32, device="cuda") for s in ((b,), (b,), (b, t)))
    lib, stream = rocm.load(), torch.cuda.Stream()
    torch.cuda.synchronize()

    def body():
        rocm.call("aljabr_rocm_set_stream", stream.cuda_stream)
        rocm.call("aljabr_rocm_set_sync_mode", 0)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
            out.fill_(POISON)
            rc = lib.aljabr_rocm_kv_tree_attention(out.data_ptr(), qd.data_ptr(), dev.ref(), 0, lens.data_ptr(), counts.data_ptr(),
                                                   up.data_ptr(), t, hkv * g, 0.0, 0, 0.0, ws[1].data_ptr(), ws[1].numel())
        rocm.call("aljabr_rocm_set_stream", None)
        rocm.call("aljabr_rocm_set_sync_mode", 1)
        assert rc == 0
        for i in (0, 1, 2, 0, 2, 1):
            for dst, src in ((lens, runs[i][0]), (counts, runs[i][1]), (up, trees[i])):
                dst.copy_(ints(src))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert np.array_equal(out.cpu().numpy(), eager[i])
        return True

    assert fresh_thread(body)


@pytest.mark.parametrize("room", [0, ROOM])
@pytest.mark.parametrize("cap", [3.4e38, 1e10, 1e-6, 1e-44])
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("t", [1, 10, 40])
def test_soft_caps_of_any_size(rocm, room, cap, dtype, t):
    """A cap far past the scores is none (4 roundings of each score for its products and tanh more than the bound without
    one); under one next to zero every key weighs the same to 2e-6."""
    host = plain.Cache(2, 1, 128, 208, 0, dtype)
    host.fill([200, 9])
    q = normal(t, 2, t, 4, 128)
    want, bound, live = plain.attention(host, q if cap > 1 else np.zeros_like(q), [200, 9])
    k = host.rows_of("k", 0, 200)[0]
    v = np.abs(host.rows_of("v", 0, 200)[0]).max()
    top = (np.abs(k) @ np.abs(q[0].reshape(-1, 128).T)).max() * 128 ** -0.5
    more = 2 * v * 4 * top * 2.0 ** -24 if cap > 1 else 2 * 2 * 1e-6 * v
    check(attend(rocm, Device(rocm, host, room), q, [200, 9], cap=cap), want, bound + more, live)


@pytest.mark.parametrize("room", [0, ROOM])
@pytest.mark.parametrize("d,t", [(64, 1), (128, 5), (256, 1), (128, 40), (256, 40), (64, 12)])
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("scale,size", [(3.4e38, 1e-39), (2.5e38, 1e-38), (1e-38, 2e37), (2e-39, 1e38), (1e30, 1e-31)])
def test_scales_at_the_ends_of_fp32(rocm, room, d, t, dtype, scale, size):
    """Queries and scales whose product alone is in range."""
    host = plain.Cache(1, 1, d, 208, 0, dtype)
    host.fill([200])
    with np.errstate(over="ignore"):
        q = normal(t, 1, t, 4, d) * np.float32(size)
    scale = float(np.float32(scale))
    want, bound, live = plain.attention(host, q, [200], scale=scale)
    got = attend(rocm, Device(rocm, host, room), q, [200], scale=scale)
    past = ~np.isfinite(q).all(-1)                                     # at 1e38 some element is infinite: its row is NaN
    assert np.isnan(got[past]).all() and np.isnan(want[past]).all()
    check(*(np.where(past[..., None], 0.0, x) for x in (got, want, bound)), live)


@pytest.mark.parametrize("room", [0, ROOM])
def test_same_call_same_bits(rocm, room):
    host = plain.Cache(2, 4, 128, 1024)
    host.fill([1024, 513])
    dev = Device(rocm, host, room)
    for t in (1, 30):
        q, parents = normal(11, 2, t, 16, 128), plain.random_parents(np.random.default_rng(1), 2, t)
        first = attend(rocm, dev, q, [1024, 513], None, parents)
        for _ in range(3):
            assert np.array_equal(first, attend(rocm, dev, q, [1024, 513], None, parents))


def test_a_sessions_cache(rocm):
    """attention_gqa's K and V are a contiguous cache of one layer: the same decode."""
    host = plain.Cache(3, 2, 128, 300)
    host.fill([300] * 3)
    dev = Device(rocm, host)
    q = normal(5, 3, 1, 8, 128)
    got = attend(rocm, dev, q, [300] * 3)
    qd, out = torch.from_numpy(q).cuda(), torch.zeros(3, 8, 1, 128, device="cuda")
    torch.cuda.synchronize()
    rocm.call("aljabr_rocm_attention_gqa", out.data_ptr(), qd.data_ptr(), dev.planes["k"].data_ptr(), dev.planes["v"].data_ptr(), None, 3, 8,
              2, 1, 300, 128, F16, 0.0, 1)
    want, bound, live = plain.attention(host, q, [300] * 3)
    check(got, want, bound, live)
    assert np.abs(out.cpu().numpy().reshape(got.shape) - got).max() <= 1e-4


def test_planes_of_a_llama_session(rocm):
    """The planes a session decoded into, described to the calls: a tree over its last rows, and the rows it accepts moved
    where the session's next step reads them."""
    from aljabr_amd.llama import LLAMA3_8B, DeviceLlama, random_weights
    cfg = dict(LLAMA3_8B, layers=2, dim=512, ffn=1024, n_heads=8, n_kv_heads=2, head_dim=64, vocab=512)
    b, steps, t, room = 3, 9, 5, 24
    model = DeviceLlama(cfg, random_weights(cfg, seed=3), max_batch=b, max_seq=room)
    k, v = model.kv_cache_ptrs()
    host = plain.Cache(b, 2, 64, room, 0, F16, 2)
    for pos in range(steps):
        model.decode(ints([7 + pos, 40 + pos, 90 + pos]), ints([pos] * b), b)

    def read():
        torch.cuda.synchronize()
        for w, at in zip("kv", (k, v)):
            plane = torch.empty(host.planes[w].size, dtype=torch.float16, device="cuda")
            rocm.call("aljabr_rocm_memcpy_d2d", plane.data_ptr(), at, 2 * plane.numel())
            rocm.call("aljabr_rocm_synchronize")
            yield w, plane.cpu().numpy().reshape(host.planes[w].shape)

    host.planes = dict(read())
    desc = rocm.KvCache(k, v, None, F16, 2, b, 2, 64, room, 0, 0)
    need = ctypes.c_size_t()
    rocm.call("aljabr_rocm_kv_cache_bytes", ctypes.byref(desc), ctypes.byref(need))
    assert need.value == 2 * model.kv_cache_elems()
    lens, parents = [steps] * b, np.array([[-1, 0, 0, 2, 1]] * b, np.int32)
    q = normal(1, b, t, 8, 64)
    qd, ld, pd, out = torch.from_numpy(q).cuda(), ints(lens), ints(parents), torch.full(q.shape, POISON, device="cuda")
    torch.cuda.synchronize()
    for layer in range(2):
        rocm.call("aljabr_rocm_kv_tree_attention", out.data_ptr(), qd.data_ptr(), ctypes.byref(desc), layer, ld.data_ptr(), None,
                  pd.data_ptr(), t, 8, 0.0, 0, 0.0, None, 0)
        torch.cuda.synchronize()
        check(out.cpu().numpy(), *plain.attention(host, q, lens, None, parents, layer=layer))
    tokens, choices = np.array([[1, 2, 3, 4, 5]] * b), np.array([[3, 0, 4, 9, 0], [2, 5, 0, 0, 8], [7, 0, 0, 0, 0]])
    outs = [torch.zeros(s, dtype=torch.int32, device="cuda") for s in ((b,), (b, t), (b,), (b,))]
    td, cd = ints(tokens), ints(choices)
    torch.cuda.synchronize()
    rocm.call("aljabr_rocm_kv_tree_accept", ctypes.byref(desc), *[o.data_ptr() for o in outs], ld.data_ptr(), None, pd.data_ptr(),
              td.data_ptr(), cd.data_ptr(), t)
    want = plain.accept(host, lens, None, parents, tokens, choices)
    assert all(np.array_equal(x.cpu().numpy(), y) for x, y in zip(outs, want)) and want[2].tolist() == [3, 3, 1]
    for w, plane in read():
        assert np.array_equal(plane, host.planes[w], equal_nan=True)
    model.decode(outs[3], outs[0], b)                                  # the next step writes behind the accepted rows
    after = dict(read())
    for i, n in enumerate(want[0]):
        assert np.array_equal(after["k"][:, i, :, :n], host.planes["k"][:, i, :, :n])
        assert not np.array_equal(after["k"][:, i, :, n], host.planes["k"][:, i, :, n])
    model.close()


# ---- accepted rows --------------------------------------------------------------------

def take(rocm, dev, lens, counts, parents, tokens, choices):
    b, t = tokens.shape
    outs = [torch.full(s, -7, dtype=torch.int32, device="cuda") for s in ((b,), (b, t), (b,), (b,))]
    args = [ints(x) for x in (lens, counts, parents, tokens, choices)]
    torch.cuda.synchronize()
    rocm.call("aljabr_rocm_kv_tree_accept", dev.ref(), *[o.data_ptr() for o in outs], *[ptr(a) for a in args], t)
    torch.cuda.synchronize()
    return [o.cpu().numpy() for o in outs]


def agreeing(rng, parents, t, share=0.8, vocab=50):
    """Tokens and choices that agree along a line, at each row with the given chance; twins among the children."""
    b = len(parents)
    tokens, choices = rng.integers(0, vocab, (b, t)), rng.integers(0, vocab, (b, t))
    for s in range(b):
        row = 0
        while rng.random() < share:
            on = [i for i in range(row + 1, t) if parents[s][i] == row]
            if not on:
                break
            row, last = int(rng.choice(on)), row
            choices[s, last] = tokens[s, row]
    return tokens, choices


@pytest.mark.parametrize("d,dtype", [(64, F16), (128, F16), (256, F32), (128, F32), (256, F16)])
@pytest.mark.parametrize("t,layers,page", [(1, 1, 0), (2, 3, 16), (8, 2, 0), (33, 1, 16), (64, 3, 0), (256, 1, 64)])
@pytest.mark.parametrize("deep", [0, 1])
def test_accept(rocm, d, dtype, t, layers, page, deep):
    b = 6
    rng = np.random.default_rng(t + d)
    parents = plain.random_parents(rng, b, t, bool(deep))
    tokens, choices = agreeing(rng, parents, t, 0.97 if deep else 0.8, 4 if t < 9 else 50)
    lens = [t, t + 9, t + 20, t + 1, t + 3, 0]
    counts = [t, t, max(t - 1, 0), 0, t, 0]
    host = plain.Cache(b, 3, d, t + 21, page, dtype, layers)
    host.fill(lens)
    dev = Device(rocm, host)
    got = take(rocm, dev, lens, counts, parents, tokens, choices)
    want = plain.accept(host, lens, counts, parents, tokens, choices)
    for x, y in zip(got, want):
        assert np.array_equal(x, y)
    check_planes(dev)


def test_accept_of_a_chain(rocm):
    """Rows of a chain are in place already: the longest prefix that agrees."""
    host = plain.Cache(3, 2, 64, 40)
    host.fill([30] * 3)
    dev = Device(rocm, host)
    tokens = np.array([[5, 6, 7, 8]] * 3)
    choices = np.array([[6, 7, 8, 9], [6, 1, 8, 9], [0, 7, 8, 9]])
    got = take(rocm, dev, [30] * 3, None, None, tokens, choices)
    assert got[0].tolist() == [30, 28, 27] and got[2].tolist() == [4, 2, 1] and got[3].tolist() == [9, 1, 0]
    assert got[1].tolist() == [[0, 1, 2, 3], [0, 1, -1, -1], [0, -1, -1, -1]]
    check_planes(dev)


def test_accept_with_numbers_that_are_no_rows(rocm):
    """Parents that are no earlier rows, all tokens alike, places and blocks that are not there, more rows than keys."""
    b, t = 5, 16
    rng = np.random.default_rng(2)
    parents = rng.integers(-3, t + 3, (b, t)).astype(np.int32)
    parents[:, 1:5] = [0, 0, 1, 3]
    parents[:, 0] = [7, -1, 2 ** 31 - 1, 0, -2 ** 31]
    tokens = np.ones((b, t), int)
    host = plain.Cache(b, 2, 128, 48, 16, F16, 2)
    host.fill([48] * b)
    host.table[1, 1], host.table[2, 2], host.table[3, :] = -1, host.s, 2 ** 31 - 1
    dev = Device(rocm, host)
    lens = [40, 30, 40, 40, 3]
    got = take(rocm, dev, lens, None, parents, tokens, tokens)
    want = plain.accept(host, lens, None, parents, tokens, tokens)
    for x, y in zip(got, want):
        assert np.array_equal(x, y)
    assert want[2].min() >= 3
    check_planes(dev)


# ---- together, as a serving program runs them ------------------------------------------

class Model:
    """One attention layer over token embeddings, in torch: enough for choices that depend on the whole context."""

    def __init__(self, vocab=97, hq=8, hkv=2, d=64, dim=96, seed=5):
        g = torch.Generator().manual_seed(seed)
        n = lambda *s: torch.randn(*s, generator=g)
        self.vocab, self.hq, self.hkv, self.d = vocab, hq, hkv, d
        self.embed, self.qkv = n(vocab, dim), (n(dim, (hq + 2 * hkv) * d) * dim ** -0.5)
        self.out = n(hq * d, vocab) * 0.3
        self.embed_d, self.qkv_d, self.out_d = (x.cuda() for x in (self.embed, self.qkv, self.out))

    def greedy(self, tokens, steps):
        """(the next tokens, the least distance of a choice to the second) in float64."""
        tokens, near = list(tokens), np.inf
        for _ in range(steps):
            x = (self.embed[tokens].double() @ self.qkv.double()).numpy().reshape(len(tokens), -1, self.d)
            turned = np.stack([plain.rotate(x[i], i, 1e4, self.d, False, None)[0] for i in range(len(tokens))])
            q, k = turned[-1, :self.hq], turned[:, self.hq:self.hq + self.hkv]
            v = x[:, self.hq + self.hkv:]
            outs = []
            for h in range(self.hq):
                s = k[:, h * self.hkv // self.hq] @ q[h] * self.d ** -0.5
                w = np.exp(s - s.max())
                outs.append(w @ v[:, h * self.hkv // self.hq] / w.sum())
            logits = np.concatenate(outs) @ self.out.double().numpy()
            top = np.sort(logits)[-2:]
            near = min(near, top[1] - top[0])
            tokens.append(int(logits.argmax()))
        return tokens, near


@pytest.mark.parametrize("page", [0, 16])
@pytest.mark.parametrize("captured", [False, True])
def test_drafted_decoding_is_greedy_decoding(rocm, page, captured):
    """Two sequences decoded with trees of 12 drafts, half of them right: append, attention, logits, argmax, accept, in one
    graph replayed each step or as calls, against decoding a token at a time in float64."""
    m, b, t, steps, dtype = Model(), 2, 12, 6, F32
    prompts = [[3, 14, 15, 92, 65, 35], [27, 18, 28]]
    host = plain.Cache(b, m.hkv, m.d, 96, page, dtype, 1)
    for w in "kv":
        host.planes[w][:] = 0
    dev = Device(rocm, host)
    want, near = zip(*(m.greedy(p, steps * 5) for p in prompts))
    assert min(near) > 1e-3                                            # far beyond what fp32 work is off by
    rng = np.random.default_rng(0)
    zeros = lambda *s, **k: torch.zeros(*s, device="cuda", **k)
    tokens, parents, angles, choices = (zeros(b, t, dtype=torch.int32) for _ in range(4))
    pos, lens, new_lens, accepted, after = (zeros(b, dtype=torch.int32) for _ in range(5))
    path = zeros(b, t, dtype=torch.int32)
    q_out, out = zeros(b, t, m.hq, m.d), zeros(b, t, m.hq, m.d)
    n = ctypes.c_size_t()
    rocm.call("aljabr_rocm_kv_tree_attention_workspace", dev.ref(), t, m.hq, ctypes.byref(n))
    ws = zeros(max(n.value, 16), dtype=torch.uint8)
    rotation = rocm.Rotation(1e4, 0, 0, None)
    row = (m.hq + 2 * m.hkv) * m.d

    def step():
        x = m.embed_d[tokens.long()].reshape(b * t, -1) @ m.qkv_d
        rocm.call("aljabr_rocm_kv_append", dev.ref(), 0, q_out.data_ptr(), x.data_ptr(), x.data_ptr() + 4 * m.hq * m.d,
                  x.data_ptr() + 4 * (m.hq + m.hkv) * m.d, pos.data_ptr(), None, angles.data_ptr(), t, m.hq, t * row, row, m.d, t * row, row,
                  m.d, F32, ctypes.byref(rotation))
        rocm.call("aljabr_rocm_kv_tree_attention", out.data_ptr(), q_out.data_ptr(), dev.ref(), 0, lens.data_ptr(), None, parents.data_ptr(),
                  t, m.hq, 0.0, 0, 0.0, ws.data_ptr(), ws.numel())
        logits = out.reshape(b * t, -1) @ m.out_d
        rocm.call("aljabr_rocm_argmax", choices.data_ptr(), logits.data_ptr(), b * t, m.vocab)
        rocm.call("aljabr_rocm_kv_tree_accept", dev.ref(), new_lens.data_ptr(), path.data_ptr(), accepted.data_ptr(), after.data_ptr(),
                  lens.data_ptr(), None, parents.data_ptr(), tokens.data_ptr(), choices.data_ptr(), t)

    s = torch.cuda.Stream()
    torch.cuda.synchronize()

    def body():
        rocm.call("aljabr_rocm_set_stream", s.cuda_stream)
        rocm.call("aljabr_rocm_set_sync_mode", 0)
        with torch.cuda.stream(s):
            step()                                                     # libraries set themselves up outside a capture
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        if captured:
            with torch.cuda.graph(graph, stream=s, capture_error_mode="thread_local"):
                step()
        # Prompts through the same calls, as chains of up to t rows.
        have = [[] for _ in range(b)]
        for i in range(b):
            p = prompts[i][:-1]
            x = (m.embed[p] @ m.qkv).reshape(1, len(p), -1, m.d).numpy()
            one = rocm.KvCache.from_buffer_copy(dev.desc)
            one.sequences = 1
            if page:
                one.block_table = dev.table.data_ptr() + 4 * i * host.per
            else:
                one.k, one.v = (dev.planes[w].data_ptr() + 4 * i * m.hkv * host.rows * m.d for w in "kv")
            kd, vd = (torch.from_numpy(np.ascontiguousarray(x[:, :, a:a + m.hkv])).cuda() for a in (m.hq, m.hq + m.hkv))
            at = ints([0])
            torch.cuda.synchronize()
            rocm.call("aljabr_rocm_kv_append", ctypes.byref(one), 0, None, None, kd.data_ptr(), vd.data_ptr(), at.data_ptr(), None, None,
                      len(p), 0, 0, 0, 0, 0, 0, 0, F32, ctypes.byref(rotation))
            torch.cuda.synchronize()
            have[i] = list(p)
        last, most = [p[-1] for p in prompts], 0
        for _ in range(steps):
            par = plain.random_parents(rng, b, t, True)
            tok = rng.integers(0, m.vocab, (b, t))
            tok[:, 0] = last
            for i in range(b):                                         # along one line the drafts are right half the time
                line = plain.line(par[i], t - 1)[::-1]
                for j, r in enumerate(line[1:], 1):
                    if rng.random() < 0.7 and len(have[i]) + j < len(want[i]):
                        tok[i, r] = want[i][len(have[i]) + j]
            depth = np.array([[len(plain.line(par[i], r)) - 1 for r in range(t)] for i in range(b)])
            start = np.array([len(h) for h in have])
            for dst, src in ((tokens, tok), (parents, par), (angles, start[:, None] + depth), (pos, start), (lens, start + t)):
                dst.copy_(ints(src))
            torch.cuda.synchronize()
            if captured:
                graph.replay()
            else:
                with torch.cuda.stream(s):
                    step()
            torch.cuda.synchronize()
            p, a, c = path.cpu().numpy(), accepted.cpu().numpy(), after.cpu().numpy()
            assert (new_lens.cpu().numpy() == start + a).all()
            for i in range(b):
                have[i] += [int(tok[i, r]) for r in p[i, :a[i]]]
                assert have[i] == want[i][:len(have[i])]
                assert int(c[i]) == want[i][len(have[i])]
            last, most = c.tolist(), max(most, int(a.max()))
        assert most >= 3
        rocm.call("aljabr_rocm_set_stream", None)
        rocm.call("aljabr_rocm_set_sync_mode", 1)
        return True

    assert fresh_thread(body)


def test_capture_without_workspace_is_refused(rocm):
    host = plain.Cache(1, 2, 128, 2048)
    host.fill([2000])
    dev, q, lens = Device(rocm, host), torch.from_numpy(normal(1, 1, 1, 8, 128)).cuda(), ints([2000])
    out = torch.zeros(1, 1, 8, 128, device="cuda")
    lib, s = rocm.load(), torch.cuda.Stream()
    torch.cuda.synchronize()

    def body():
        rocm.call("aljabr_rocm_set_stream", s.cuda_stream)
        rocm.call("aljabr_rocm_set_sync_mode", 0)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s, capture_error_mode="thread_local"):
            out.add_(0)
            rc = lib.aljabr_rocm_kv_tree_attention(out.data_ptr(), q.data_ptr(), dev.ref(), 0, lens.data_ptr(), None, None, 1, 8, 0.0, 0,
                                                   0.0, None, 0)
        rocm.call("aljabr_rocm_set_stream", None)
        rocm.call("aljabr_rocm_set_sync_mode", 1)
        return rc, scratch_held(rocm)

    assert fresh_thread(body) == (-4, 0)


def test_two_streams_at_once(rocm):
    """Calls of two threads on streams of their own share nothing but the cache they read."""
    host = plain.Cache(2, 4, 128, 1024)
    host.fill([1024, 900])
    dev = Device(rocm, host)
    qs = [normal(20 + i, 2, t, 16, 128) for i, t in enumerate((1, 20))]
    want = [attend(rocm, dev, q, [1024, 900]) for q in qs]

    def work(i):
        return [attend(rocm, dev, qs[i], [1024, 900]) for _ in range(6)]

    import concurrent.futures as cf
    with cf.ThreadPoolExecutor(2) as pool:
        for i, outs in enumerate(pool.map(work, (0, 1))):
            for got in outs:
                assert np.array_equal(got, want[i])
