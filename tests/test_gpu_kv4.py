"""The 4-bit KV cache on the GPU: rows written and read bit for bit, attention
against float64 within the bound that ``kv4_plain.attention`` derives, bad
pages, garbage past a sequence's end, capture into graphs, several streams."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import kv4_plain as plain
from conftest import fresh_thread, scratch_held

pytestmark = pytest.mark.gpu

F32, F16 = 0, 1
POISON = -77.0


class Device:
    """A host cache's planes on the GPU and the description the calls take."""

    def __init__(self, rocm, host):
        put = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
        self.host, self.abi = host, rocm
        self.codes = {w: put(host.codes[w]) for w in "kv"}
        self.scales = {w: put(host.scales[w]) for w in "kv"}
        self.table = None if host.table is None else put(host.table)
        self.desc = rocm.Kv4Cache(self.codes["k"].data_ptr(), self.scales["k"].data_ptr(), self.codes["v"].data_ptr(),
                                  self.scales["v"].data_ptr(), None if self.table is None else self.table.data_ptr(),
                                  host.seqs, host.heads, host.d, host.rows, host.s if host.page else 0,
                                  host.per if host.page else 0)
        torch.cuda.synchronize()

    def ref(self):
        return ctypes.byref(self.desc)

    def planes_equal(self):
        torch.cuda.synchronize()
        for w in "kv":
            assert np.array_equal(self.codes[w].cpu().numpy(), self.host.codes[w])
            assert np.array_equal(self.scales[w].cpu().numpy(), self.host.scales[w], equal_nan=True)


def ints(x):
    return None if x is None else torch.tensor(np.asarray(x), dtype=torch.int32).cuda()


def ptr(t):
    return None if t is None else t.data_ptr()


def attend(rocm, dev, q, lens, counts=None, causal=1, window=0, cap=0.0, scale=0.0, workspace=None):
    B, T, Hq, _ = q.shape
    qd, ld, cd = torch.from_numpy(q).cuda(), ints(lens), ints(counts)
    out = torch.full(q.shape, POISON, device="cuda")
    torch.cuda.synchronize()
    rocm.call("aljabr_rocm_kv4_attention", out.data_ptr(), qd.data_ptr(), dev.ref(), ld.data_ptr(), ptr(cd), T, Hq, scale,
              causal, window, cap, ptr(workspace), 0 if workspace is None else workspace.numel())
    torch.cuda.synchronize()
    return out.cpu().numpy()


def check(got, want, bound, live):
    assert (got[~live] == POISON).all(), "rows behind a sequence's last were written"
    err = np.abs(got.astype(np.float64) - want)[live]
    assert (err <= bound[live] + 1e-30).all(), (np.nanmax(err), np.nanmax(err / (bound[live] + 1e-30)), np.isnan(err).sum())


# ---- rows --------------------------------------------------------------------------

def rows(seed, b, t, h, d):
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((b, t, h, d)) * np.exp(rng.uniform(-3, 3, (b, t, h, 1)))).astype(np.float32)
    flat = x.reshape(-1, 32)
    special = [np.zeros(32), np.where(np.arange(32) == 7, 3.0, 0), np.arange(32) - 15.5, -(np.arange(32) - 15.5),
               (rng.integers(-16, 17, 32) / 2.0), np.full(32, -1e-7), np.linspace(-3e-6, 2e-6, 32), np.linspace(-1e30, 7e29, 32),
               np.full(32, 70000.0), np.linspace(-65280, 65279, 32), np.full(32, 5e-324), np.linspace(1, 2, 32),
               np.where(np.arange(32) % 2, 8.0, -8.0), np.where(np.arange(32) == 31, np.inf, 1.0),
               np.where(np.arange(32) == 0, np.nan, 1.0), np.full(32, -0.0), 1 + np.arange(32) * 2.0 ** -23]
    for i, s in enumerate(special):
        flat[(i * 5 + seed) % len(flat)] = s
    return x


def lay_out(x, layout):
    """A float array [B, T, H, D] as (device tensor, pointer offset in elements, strides)."""
    b, t, h, d = x.shape
    if layout == "dense":
        return x.copy(), 0, (0, 0, 0)
    if layout == "heads":
        return np.ascontiguousarray(x.transpose(0, 2, 1, 3)), 0, (h * t * d, d, t * d)
    pad = 5 if layout == "odd" else 8                       # odd: rows off the wide loads' alignment
    row = h * d + pad
    out = np.full((b, t, row), 9.0, x.dtype)
    out[:, :, pad - 1 if layout == "odd" else 4:][:, :, :h * d] = x.reshape(b, t, -1)
    return out, pad - 1 if layout == "odd" else 4, (t * row, row, d)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("t,page,dtype,layout", [(1, 0, F32, "dense"), (1, 16, F16, "heads"), (5, 48, F32, "odd"),
                                                 (15, 0, F16, "odd"), (16, 32, F32, "row"), (37, 16, F32, "heads"),
                                                 (70, 0, F16, "dense"), (33, 64, F16, "row")])
@pytest.mark.parametrize("h", [1, 3])
def test_write_and_read_bit_for_bit(rocm, d, t, page, dtype, layout, h):
    b, np_t = 3, np.float32 if dtype == F32 else np.float16
    with np.errstate(over="ignore"):
        k, v = (rows(s, b, t, h, d).astype(np_t) for s in (1, 2))
    host = plain.Cache(b, h, d, 96, page)
    dev = Device(rocm, host)
    start, counts = [0, 11, 96 - t], [t, max(t - 2, 0), t]
    for s in range(b):
        for i in range(counts[s]):
            for w, x in (("k", k), ("v", v)):
                host.write(w, s, start[s] + i, x[s, i])
    bufs = [lay_out(x, layout) for x in (k, v)]
    devs = [torch.from_numpy(x[0]).cuda() for x in bufs]
    off, strides = bufs[0][1] * np_t().itemsize, bufs[0][2]
    pos, cnt = ints(start), ints(counts)
    torch.cuda.synchronize()
    rocm.call("aljabr_rocm_kv4_write", dev.ref(), devs[0].data_ptr() + off, devs[1].data_ptr() + off, pos.data_ptr(),
              cnt.data_ptr(), t, *strides, dtype)
    dev.planes_equal()
    for out_t in (F32, F16):
        outs = [torch.full((b, t, h, d), POISON, device="cuda", dtype=torch.float32 if out_t == F32 else torch.float16)
                for _ in "kv"]
        torch.cuda.synchronize()
        rocm.call("aljabr_rocm_kv4_read", outs[0].data_ptr(), outs[1].data_ptr(), dev.ref(), pos.data_ptr(), cnt.data_ptr(), t,
                  0, 0, 0, out_t)
        for w, o in zip("kv", outs):
            got = o.cpu().numpy()
            for s in range(b):
                want, _ = host.rows_of(w, s, start[s] + counts[s])
                assert np.array_equal(got[s, :counts[s]].astype(np.float64),
                                      want[:, start[s]:].transpose(1, 0, 2).astype(np.float64), equal_nan=True)
                assert (got[s, counts[s]:] == POISON).all()


@pytest.mark.parametrize("layout", ["heads", "odd"])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_read_into_strided_rows(rocm, layout, dtype):
    b, t, h, d = 2, 21, 3, 128
    np_t = np.float32 if dtype == F32 else np.float16
    host = plain.Cache(b, h, d, 64, 16)
    host.fill([30, 40])
    dev = Device(rocm, host)
    blank, off, strides = lay_out(np.full((b, t, h, d), POISON, np_t), layout)
    outs = [torch.from_numpy(blank).cuda() for _ in "kv"]
    pos = ints([3, 19])
    torch.cuda.synchronize()
    rocm.call("aljabr_rocm_kv4_read", outs[0].data_ptr() + off * np_t().itemsize, outs[1].data_ptr() + off * np_t().itemsize,
              dev.ref(), pos.data_ptr(), None, t, *strides, dtype)
    for w, o in zip("kv", outs):
        want = np.stack([host.rows_of(w, s, p + t)[0][:, p:].transpose(1, 0, 2) for s, p in ((0, 3), (1, 19))]).astype(np_t)
        assert np.array_equal(o.cpu().numpy(), lay_out(want, layout)[0])


def test_rows_that_the_cache_does_not_have(rocm):
    b, t, h, d = 4, 8, 2, 64
    host = plain.Cache(b, h, d, 48, 16)
    host.fill([48, 48, 48, 48])
    host.table[0, 1], host.table[1, 0], host.table[2, 2] = -1, host.s, 2 ** 31 - 1
    dev = Device(rocm, host)
    x = rows(5, b, t, h, d)
    start = [12, 12, -3, 44]
    for s in range(b):
        for i in range(t):
            host.write("k", s, start[s] + i, x[s, i])
            host.write("v", s, start[s] + i, x[s, i])
    xd, pos = torch.from_numpy(x).cuda(), ints(start)
    outs = [torch.full((b, t, h, d), POISON, device="cuda") for _ in "kv"]
    torch.cuda.synchronize()
    rocm.call("aljabr_rocm_kv4_write", dev.ref(), xd.data_ptr(), xd.data_ptr(), pos.data_ptr(), None, t, 0, 0, 0, F32)
    dev.planes_equal()
    rocm.call("aljabr_rocm_kv4_read", outs[0].data_ptr(), outs[1].data_ptr(), dev.ref(), pos.data_ptr(), None, t, 0, 0, 0, F32)
    got = outs[0].cpu().numpy()
    for s in range(b):
        for i in range(t):
            at = host.at(s, start[s] + i)
            want = 0.0 if at is None else plain.decode(host.codes["k"][at[0], :, at[1]], host.scales["k"][at[0], :, :, at[1]])
            assert np.array_equal(got[s, i].astype(np.float64), np.broadcast_to(want, (h, d)).astype(np.float64), equal_nan=True)


def test_one_of_k_and_v(rocm):
    b, t, h, d = 1, 3, 2, 128
    host = plain.Cache(b, h, d, 16)
    dev = Device(rocm, host)
    x = rows(6, b, t, h, d)
    xd, pos = torch.from_numpy(x).cuda(), ints([2])
    torch.cuda.synchronize()
    rocm.call("aljabr_rocm_kv4_write", dev.ref(), None, xd.data_ptr(), pos.data_ptr(), None, t, 0, 0, 0, F32)
    for i in range(t):
        host.write("v", 0, 2 + i, x[0, i])
    dev.planes_equal()
    rocm.call("aljabr_rocm_kv4_write", dev.ref(), xd.data_ptr(), None, pos.data_ptr(), None, t, 0, 0, 0, F32)
    for i in range(t):
        host.write("k", 0, 2 + i, x[0, i])
    dev.planes_equal()
    out = torch.full((b, t, h, d), POISON, device="cuda")
    torch.cuda.synchronize()
    rocm.call("aljabr_rocm_kv4_read", None, out.data_ptr(), dev.ref(), pos.data_ptr(), None, t, 0, 0, 0, F32)
    assert np.array_equal(out.cpu().numpy()[0], host.rows_of("v", 0, 5)[0][:, 2:].transpose(1, 0, 2).astype(np.float32), equal_nan=True)


# ---- attention ---------------------------------------------------------------------

def query(seed, b, t, hq, d):
    return np.random.default_rng(seed).standard_normal((b, t, hq, d)).astype(np.float32)


SHAPES = [(1, 1), (8, 4), (4, 8), (2, 3), (1, 16), (3, 7)]           # (KV heads, query heads of each)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hkv,g", SHAPES)
@pytest.mark.parametrize("page", [0, 16, 48])
def test_decode(rocm, d, hkv, g, page):
    lens = [1, 33, 200, 0]
    host = plain.Cache(4, hkv, d, 208, page)
    host.fill(lens)
    q = query(d + g, 4, 1, hkv * g, d)
    got = attend(rocm, Device(rocm, host), q, lens)
    check(got, *plain.attention(host, q, lens))
    assert not got[3].any()                                           # no key: zeros


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 127, 128, 129, 255, 257, 511, 1000, 2047])
def test_lengths(rocm, n):
    host = plain.Cache(1, 2, 128, 2048)
    host.fill([n], seed=n)
    q = query(n, 1, 1, 8, 128)
    check(attend(rocm, Device(rocm, host), q, [n]), *plain.attention(host, q, [n]))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("t,hkv,g", [(2, 2, 4), (5, 2, 2), (8, 1, 8), (9, 2, 1), (17, 2, 4), (40, 1, 3), (70, 2, 2)])
@pytest.mark.parametrize("causal,window,cap", [(1, 0, 0.0), (0, 0, 0.0), (1, 20, 0.0), (0, 24, 0.0), (1, 40, 5.0), (1, 1, 0.0)])
def test_several_rows(rocm, d, t, hkv, g, causal, window, cap):
    lens, counts = [t, 100, 3, 150], [t, max(t - 3, 1), t, 0]         # the third: more rows than keys
    host = plain.Cache(4, hkv, d, 160, 16 if t % 2 else 0)
    host.fill(lens)
    q = query(t, 4, t, hkv * g, d)
    got = attend(rocm, Device(rocm, host), q, lens, counts, causal, window, cap)
    check(got, *plain.attention(host, q, lens, counts, bool(causal), window, cap))


def test_scale_and_large_scores(rocm):
    host = plain.Cache(1, 2, 128, 304)
    host.fill([300])
    dev = Device(rocm, host)
    for scale, size in ((0.5, 1.0), (2.0, 30.0), (1e-3, 1e-20), (1e-4, 1e6)):
        q = query(3, 1, 2, 4, 128) * np.float32(size)
        check(attend(rocm, dev, q, [300], scale=scale), *plain.attention(host, q, [300], scale=scale))


def test_scales_of_any_fp16_number(rocm):
    """Scales that kv4_write would not make: values are the products rounded to fp16."""
    host = plain.Cache(1, 2, 128, 112)
    rng = np.random.default_rng(9)
    for w in "kv":
        host.codes[w][:] = rng.integers(0, 256, host.codes[w].shape)
        host.scales[w][:] = (rng.standard_normal(host.scales[w].shape) * 0.2).astype(np.float16)
    q = query(4, 1, 3, 8, 128)
    dev = Device(rocm, host)
    check(attend(rocm, dev, q, [101]), *plain.attention(host, q, [101]))
    out = torch.empty(1, 112, 2, 128, device="cuda", dtype=torch.float16)
    pos = ints([0])
    torch.cuda.synchronize()
    rocm.call("aljabr_rocm_kv4_read", out.data_ptr(), None, dev.ref(), pos.data_ptr(), None, 112, 0, 0, 0, F16)
    assert np.array_equal(out.cpu().numpy()[0].transpose(1, 0, 2), host.rows_of("k", 0, 112)[0])


def test_small_values(rocm):
    """Scales down in fp16's subnormal numbers."""
    host = plain.Cache(1, 1, 128, 64)
    rng = np.random.default_rng(2)
    for w in "kv":
        for pos in range(64):
            host.write(w, 0, pos, (rng.standard_normal((1, 128)) * 2e-5).astype(np.float32))
    q = query(5, 1, 1, 4, 128) * np.float32(3e4)
    check(attend(rocm, Device(rocm, host), q, [64]), *plain.attention(host, q, [64]))


@pytest.mark.parametrize("t", [1, 6, 40])
def test_bad_blocks_hold_no_keys(rocm, t):
    lens = [90, 90, 90, 20]
    host = plain.Cache(4, 2, 128, 96, 16)
    host.fill(lens)
    host.table[0, 2], host.table[1, 0], host.table[1, 5], host.table[3, :] = -1, host.s, 2 ** 31 - 1, -5
    q = query(6, 4, t, 8, 128)
    got = attend(rocm, Device(rocm, host), q, lens)
    check(got, *plain.attention(host, q, lens))
    assert not got[3].any()


def test_lengths_past_the_cache_are_clamped(rocm):
    host = plain.Cache(2, 2, 64, 32)
    host.fill([32, 32])
    q = query(7, 2, 1, 4, 64)
    got = attend(rocm, Device(rocm, host), q, [2 ** 31 - 1, -7])
    want, bound, live = plain.attention(host, q, [32, 0])
    check(got, want, bound, live)


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("t", [4, 40])
def test_a_value_that_is_not_finite_reaches_only_rows_that_see_it(rocm, which, t):
    host = plain.Cache(1, 2, 128, 128)
    host.fill([100])
    q = query(8, 1, t, 8, 128)
    want, bound, live = plain.attention(host, q, [100])
    bad = 98                                                           # seen by the last two rows
    x = np.random.default_rng(0).standard_normal((2, 128)).astype(np.float32)
    x[1, 37] = np.nan                                                  # one block of one head
    host.write(which, 0, bad, x)
    got = attend(rocm, Device(rocm, host), q, [100])
    check(got[:, :t - 2], want[:, :t - 2], bound[:, :t - 2], live[:, :t - 2])
    want2, bound2, _ = plain.attention(host, q, [100])
    assert np.array_equal(np.isnan(got), np.isnan(want2))
    ok = ~np.isnan(want2)
    assert (np.abs(got - want2)[ok] <= bound2[ok]).all()


def test_window_leaves_nan_behind(rocm):
    host = plain.Cache(1, 1, 64, 128)
    host.fill([120])
    host.write("v", 0, 70, np.full((1, 64), np.nan, np.float32))       # outside the windows of all rows but the first
    q = query(9, 1, 3, 4, 64)
    got = attend(rocm, Device(rocm, host), q, [120], window=48)        # rows at 117..119 see 70.., 71.., 72..
    want, bound, _ = plain.attention(host, q, [120], window=48)
    assert np.isnan(got[0, 0]).all() and np.isnan(want[0, 0]).all()
    check(got[:, 1:], want[:, 1:], bound[:, 1:], np.ones((1, 2), bool))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("t", [1, 6, 40])
@pytest.mark.parametrize("scale", [8190.0, 30000.0, -65504.0, np.inf])
def test_scales_past_fp16_outside_the_window(rocm, d, t, scale):
    """Finite scales whose values overflow, among keys of the first tiles that no row sees."""
    host = plain.Cache(1, 2, d, 208)
    host.fill([200])
    q = query(d, 1, t, 8, d)
    want = plain.attention(host, q, [200], window=48)
    first = 200 - t - 48 + 1                                           # the first key that a row sees
    for w in "kv":
        host.codes[w][:, :, :first] = np.random.default_rng(t).integers(0, 256, host.codes[w][:, :, :first].shape)
        host.scales[w][..., :first] = scale
        host.scales[w][..., 200:] = scale                              # and past the end
    check(attend(rocm, Device(rocm, host), q, [200], window=48), *want)


@pytest.mark.parametrize("t", [1, 20])
def test_workspace_of_any_size(rocm, t):
    host = plain.Cache(2, 2, 128, 1024, 32)
    lens = [1000, 700]
    host.fill(lens)
    dev = Device(rocm, host)
    q = query(10, 2, t, 8, 128)
    want = plain.attention(host, q, lens)
    n = ctypes.c_size_t()
    rocm.call("aljabr_rocm_kv4_attention_workspace", dev.ref(), t, 8, ctypes.byref(n))
    assert n.value > 0
    for size in (n.value, n.value // 2, n.value // 3, 16, 0):
        ws = torch.full((max(size, 16) + 64,), 0xCD, dtype=torch.uint8, device="cuda")
        got = attend(rocm, dev, q, lens, workspace=ws[:size] if size else None)
        check(got, *want)
        assert (ws[size:] == 0xCD).all()
    check(attend(rocm, dev, q, lens), *want)


@pytest.mark.parametrize("t,g", [(1, 4), (3, 8), (20, 4)])
@pytest.mark.parametrize("b,page", [(65, 0), (130, 16)])
def test_many_uneven_sequences(rocm, b, page, t, g):
    """More sequences than a wave has lanes, from no key to all of them."""
    rng = np.random.default_rng(b + t)
    lens = rng.integers(0, 200, b)
    lens[3], lens[64], lens[b - 1] = 200, 200, 1
    counts = rng.integers(0, t + 1, b)
    host = plain.Cache(b, 1, 64, 208, page)
    host.fill(lens)
    q = query(b, b, t, g, 64)
    got = attend(rocm, Device(rocm, host), q, lens, counts)
    check(got, *plain.attention(host, q, lens, counts))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("g", [33, 64, 130])
def test_one_token_of_many_heads(rocm, d, g):
    """Groups of more heads than the split kernel stacks."""
    lens = [500, 31, 0]
    host = plain.Cache(3, 1, d, 512)
    host.fill(lens)
    q = query(g, 3, 1, g, d)
    got = attend(rocm, Device(rocm, host), q, lens)
    check(got, *plain.attention(host, q, lens))


def test_windows_of_any_size(rocm):
    host = plain.Cache(2, 2, 64, 64)
    host.fill([40, 2])
    dev = Device(rocm, host)
    for t in (1, 5, 40):
        q = query(t, 2, t, 4, 64)
        for causal in (1, 0):
            for window in (-3, 1, 2 ** 31 - 1):
                check(attend(rocm, dev, q, [40, 2], causal=causal, window=window),
                      *plain.attention(host, q, [40, 2], causal=bool(causal), window=window))


def test_prompt_of_more_rows_than_a_grid_dimension(rocm):
    n, d = 70000, 64
    host = plain.Cache(1, 1, d, 70016)
    host.codes["k"][:], host.codes["v"][:] = (np.random.default_rng(i).integers(0, 256, host.codes["k"].shape) for i in (1, 2))
    for w in "kv":
        host.scales[w][:] = np.float16(0.25)
    dev = Device(rocm, host)
    q = query(1, 1, n, 1, d)
    got = attend(rocm, dev, q, [n], window=40)
    for at in (0, 65535, 65536, n - 1):                               # four rows, each as the last of a shorter sequence
        want, bound, live = plain.attention(host, q[:, at:at + 1], [at + 1], window=40)
        check(got[:, at:at + 1], want, bound, live)
    assert np.isfinite(got).all()


@pytest.mark.parametrize("paged", [0, 1])
@pytest.mark.parametrize("t,g", [(1, 2), (5, 8)])
def test_planes_past_32_bits(rocm, paged, t, g):
    """Rows at the end of planes of 8 GiB, seen through a window."""
    h, d, n, seen = 2, 256, 1 << 25, 80
    rows, blocks = (16, n // 16) if paged else (n, 1)
    small = plain.Cache(1, h, d, 96)                                   # the last rows alone
    codes = {w: torch.empty(blocks * h * rows * d // 2, dtype=torch.uint8, device="cuda") for w in "kv"}
    scales = {w: torch.empty(blocks * h * rows * d // 32, dtype=torch.float16, device="cuda") for w in "kv"}
    table = torch.arange(n // 16, dtype=torch.int32, device="cuda") if paged else None
    desc = rocm.Kv4Cache(codes["k"].data_ptr(), scales["k"].data_ptr(), codes["v"].data_ptr(), scales["v"].data_ptr(), ptr(table),
                         1, h, d, rows, blocks if paged else 0, n // 16 if paged else 0)
    need, sc = ctypes.c_size_t(), ctypes.c_size_t()
    rocm.call("aljabr_rocm_kv4_cache_bytes", ctypes.byref(desc), ctypes.byref(need), ctypes.byref(sc))
    assert need.value == codes["k"].numel() and sc.value == 2 * scales["k"].numel()
    x = np.random.default_rng(t).standard_normal((2, seen, h, d)).astype(np.float32)
    for i in range(seen):
        small.write("k", 0, i, x[0, i])
        small.write("v", 0, i, x[1, i])
    xd, pos, lens = torch.from_numpy(x).cuda(), ints([n - seen]), ints([n])
    back = torch.empty(1, seen, h, d, device="cuda")
    torch.cuda.synchronize()
    rocm.call("aljabr_rocm_kv4_write", ctypes.byref(desc), xd[0].data_ptr(), xd[1].data_ptr(), pos.data_ptr(), None, seen, 0, 0, 0,
              F32)
    rocm.call("aljabr_rocm_kv4_read", None, back.data_ptr(), ctypes.byref(desc), pos.data_ptr(), None, seen, 0, 0, 0, F32)
    assert np.array_equal(back[0].cpu().numpy(), small.rows_of("v", 0, seen)[0].transpose(1, 0, 2).astype(np.float32))
    q = query(2, 1, t, h * g, d)
    qd, out = torch.from_numpy(q).cuda(), torch.full(q.shape, POISON, device="cuda")
    torch.cuda.synchronize()
    rocm.call("aljabr_rocm_kv4_attention", out.data_ptr(), qd.data_ptr(), ctypes.byref(desc), lens.data_ptr(), None, t, h * g, 0.0, 1,
              64, 0.0, None, 0)
    check(out.cpu().numpy(), *plain.attention(small, q, [seen], window=64))


def test_same_call_same_bits(rocm):
    host = plain.Cache(2, 4, 128, 1024)
    host.fill([1024, 513])
    dev = Device(rocm, host)
    for t in (1, 30):
        q = query(11, 2, t, 16, 128)
        first = attend(rocm, dev, q, [1024, 513])
        for _ in range(3):
            assert np.array_equal(first, attend(rocm, dev, q, [1024, 513]))


# ---- together, as a serving program runs them ------------------------------------------

def test_capture_without_workspace_is_refused(rocm):
    host = plain.Cache(1, 2, 128, 2048)
    host.fill([2000])
    dev, q, lens = Device(rocm, host), torch.from_numpy(query(1, 1, 1, 8, 128)).cuda(), ints([2000])
    out = torch.zeros(1, 1, 8, 128, device="cuda")
    lib, s = rocm.load(), torch.cuda.Stream()
    torch.cuda.synchronize()

    def body():
        rocm.call("aljabr_rocm_set_stream", s.cuda_stream)
        rocm.call("aljabr_rocm_set_sync_mode", 0)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s, capture_error_mode="thread_local"):
            out.add_(0)
            rc = lib.aljabr_rocm_kv4_attention(out.data_ptr(), q.data_ptr(), dev.ref(), lens.data_ptr(), None, 1, 8, 0.0, 1, 0,
                                               0.0, None, 0)
        rocm.call("aljabr_rocm_set_stream", None)
        rocm.call("aljabr_rocm_set_sync_mode", 1)
        return rc

    assert fresh_thread(body) == -4


@pytest.mark.parametrize("t", [1, 12])
def test_captured_steps_write_and_attend(rocm, t):
    """Write, attend and read back in one graph, replayed while the cache grows, against eager calls and float64."""
    b, hkv, g, d, page, cap = 3, 2, 4, 128, 16, 256
    steps = 4
    host = plain.Cache(b, hkv, d, cap, page)
    start = [100, 3, 37]
    host.fill(start)
    dev = Device(rocm, host)
    pos, lens = ints(start), ints([s + t for s in start])
    k, v, q = (torch.empty(b, t, n, d, device="cuda") for n in (hkv, hkv, hkv * g))
    out, back = torch.zeros(b, t, hkv * g, d, device="cuda"), torch.zeros(b, t, hkv, d, device="cuda")
    n = ctypes.c_size_t()
    rocm.call("aljabr_rocm_kv4_attention_workspace", dev.ref(), t, hkv * g, ctypes.byref(n))
    ws = torch.zeros(max(n.value, 16), dtype=torch.uint8, device="cuda")

    def step():
        rocm.call("aljabr_rocm_kv4_write", dev.ref(), k.data_ptr(), v.data_ptr(), pos.data_ptr(), None, t, 0, 0, 0, F32)
        rocm.call("aljabr_rocm_kv4_attention", out.data_ptr(), q.data_ptr(), dev.ref(), lens.data_ptr(), None, t, hkv * g, 0.0,
                  1, 0, 0.0, ws.data_ptr(), ws.numel())
        rocm.call("aljabr_rocm_kv4_read", back.data_ptr(), None, dev.ref(), pos.data_ptr(), None, t, 0, 0, 0, F32)

    s = torch.cuda.Stream()
    torch.cuda.synchronize()

    def body():
        rocm.call("aljabr_rocm_set_stream", s.cuda_stream)
        rocm.call("aljabr_rocm_set_sync_mode", 0)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s, capture_error_mode="thread_local"):
            step()
        assert scratch_held(rocm) == 0
        at = list(start)
        for i in range(steps):
            rng = np.random.default_rng(50 + i)
            kh, vh = (rng.standard_normal((b, t, hkv, d)).astype(np.float32) for _ in "kv")
            qh = rng.standard_normal((b, t, hkv * g, d)).astype(np.float32)
            for dst, src in ((k, kh), (v, vh), (q, qh)):
                dst.copy_(torch.from_numpy(src))
            pos.copy_(ints(at))
            lens.copy_(ints([a + t for a in at]))
            out.fill_(POISON)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for j in range(b):
                for r in range(t):
                    host.write("k", j, at[j] + r, kh[j, r])
                    host.write("v", j, at[j] + r, vh[j, r])
            dev.planes_equal()
            got = out.cpu().numpy()
            check(got, *plain.attention(host, qh, [a + t for a in at]))
            for j in range(b):
                assert np.array_equal(back[j].cpu().numpy(),
                                      host.rows_of("k", j, at[j] + t)[0][:, at[j]:].transpose(1, 0, 2).astype(np.float32))
            with torch.cuda.stream(s):
                out.fill_(POISON)
            step()                                                     # eager, between the replays
            torch.cuda.synchronize()
            assert np.array_equal(got, out.cpu().numpy())
            at = [a + t for a in at]
        rocm.call("aljabr_rocm_set_stream", None)
        rocm.call("aljabr_rocm_set_sync_mode", 1)
        return True

    assert fresh_thread(body)


def test_two_streams_at_once(rocm):
    """Calls of two threads on streams of their own share nothing but the cache they read."""
    host = plain.Cache(2, 4, 128, 1024)
    host.fill([1024, 900])
    dev = Device(rocm, host)
    qs = [query(20 + i, 2, t, 16, 128) for i, t in enumerate((1, 20))]
    want = [attend(rocm, dev, q, [1024, 900]) for q in qs]

    def work(i):
        return [attend(rocm, dev, qs[i], [1024, 900]) for _ in range(6)]

    import concurrent.futures as cf
    with cf.ThreadPoolExecutor(2) as pool:
        for i, outs in enumerate(pool.map(work, (0, 1))):
            for got in outs:
                assert np.array_equal(got, want[i])


def workspace_bytes(rocm, dev, t, hq):
    n = ctypes.c_size_t()
    rocm.call("aljabr_rocm_kv4_attention_workspace", dev.ref(), t, hq, ctypes.byref(n))
    return n.value


@pytest.mark.parametrize("d,cap,t,g", [(64, 128, 1, 4), (128, 128, 5, 4), (128, 128, 20, 4), (256, 64, 1, 2), (256, 128, 40, 1)])
def test_caches_of_one_chunk_take_no_scratch(rocm, d, cap, t, g):
    """Sequences too short to be split: no partials, so a call under capture needs no workspace."""
    b = 7
    lens = [cap, 1, 33, 0, cap - 1, 64, 17]
    host = plain.Cache(b, 2, d, cap, 16)
    host.fill(lens)
    dev, q = Device(rocm, host), query(d + t, b, t, 2 * g, d)
    assert workspace_bytes(rocm, dev, t, 2 * g) == 0
    want = plain.attention(host, q, lens)
    qd, ld, out = torch.from_numpy(q).cuda(), ints(lens), torch.zeros(b, t, 2 * g, d, device="cuda")
    s = torch.cuda.Stream()
    torch.cuda.synchronize()

    def body():
        rocm.call("aljabr_rocm_set_stream", s.cuda_stream)
        rocm.call("aljabr_rocm_set_sync_mode", 0)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s, capture_error_mode="thread_local"):
            rocm.call("aljabr_rocm_kv4_attention", out.data_ptr(), qd.data_ptr(), dev.ref(), ld.data_ptr(), None, t, 2 * g, 0.0, 1,
                      0, 0.0, None, 0)
        for _ in range(3):
            out.fill_(POISON)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            check(out.cpu().numpy(), *want)
        held = scratch_held(rocm)
        rocm.call("aljabr_rocm_set_stream", None)
        rocm.call("aljabr_rocm_set_sync_mode", 1)
        return held

    assert fresh_thread(body) == 0


def scratch_test(rocm, b, t, hkv, g, d, lens, counts=None, page=0):
    """A call on exactly the workspace that was asked for, on half and a third of it; nothing past it is written."""
    host = plain.Cache(b, hkv, d, -(-max(lens) // 16) * 16, page)
    host.fill(lens)
    dev, q = Device(rocm, host), query(b + t, b, t, hkv * g, d)
    size = workspace_bytes(rocm, dev, t, hkv * g)
    assert size > 0
    want = plain.attention(host, q, lens, counts)
    for part in (1, 2, 3):
        ws = torch.full((size + 4096,), 0xCD, dtype=torch.uint8, device="cuda")
        check(attend(rocm, dev, q, lens, counts, workspace=ws[:size // part]), *want)
        assert (ws[size // part:] == 0xCD).all()


@pytest.mark.parametrize("d,t,g", [(64, 1, 3), (128, 1, 4), (128, 12, 4), (256, 2, 2)])
@pytest.mark.parametrize("page", [0, 32])
def test_workspace_of_uneven_batches(rocm, d, t, g, page):
    """A few long sequences among many short ones, in several groups of 64: only the long ones are split."""
    b = 150
    lens = [20 + 3 * (i % 7) for i in range(b)]
    for i, n in ((0, 700), (63, 1100), (64, 900), (100, 0), (127, 800), (128, 1500), (149, 1024)):
        lens[i] = n
    scratch_test(rocm, b, t, 1, g, d, lens, page=page)


def test_workspace_of_an_even_batch(rocm):
    scratch_test(rocm, 5, 1, 2, 4, 128, [900] * 5)


@pytest.mark.parametrize("b,t,hkv,g,d,block", [(64, 256, 8, 4, 128, 128), (64, 32, 8, 2, 64, 128), (1024, 1, 1, 8, 128, 8),
                                               (4096, 1, 8, 4, 256, 8)])
def test_workspace_grows_with_the_chunks_not_the_batch(rocm, b, t, hkv, g, d, block):
    """Partials of twice the chunks that fill the chip, and a first chunk and number for each sequence."""
    desc = rocm.Kv4Cache(0x10000, 0x20000, 0x30000, 0x40000, None, b, hkv, d, 4096, 0, 0)
    n = ctypes.c_size_t()
    rocm.call("aljabr_rocm_kv4_attention_workspace", ctypes.byref(desc), t, hkv * g, ctypes.byref(n))
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    groups = -(-t * g // block)
    assert n.value <= 2 * 3 * cus * block * (d + 2) * 4 + 8 * hkv * groups * b


@pytest.mark.parametrize("d,t", [(64, 1), (128, 20), (256, 3)])
@pytest.mark.parametrize("nbytes", [0, 8, 1000])
def test_a_workspace_too_small_to_split_with(rocm, d, t, nbytes):
    """A pointer with (next to) no bytes behind it: one chunk a sequence, and the stream's scratch stays untouched."""
    lens = [700, 31, 0]
    host = plain.Cache(3, 2, d, 704, 16)
    host.fill(lens)
    dev, q = Device(rocm, host), query(t, 3, t, 8, d)
    qd, ld, out = torch.from_numpy(q).cuda(), ints(lens), torch.full(q.shape, POISON, device="cuda")
    ws = torch.full((4096,), 0xCD, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()

    def body():
        rocm.call("aljabr_rocm_kv4_attention", out.data_ptr(), qd.data_ptr(), dev.ref(), ld.data_ptr(), None, t, 8, 0.0, 1, 0, 0.0,
                  ws.data_ptr(), nbytes)
        return scratch_held(rocm)

    assert fresh_thread(body) == 0
    check(out.cpu().numpy(), *plain.attention(host, q, lens))
    assert (ws == 0xCD).all()


def test_merge_of_more_rows_than_a_launch_has_lanes(rocm):
    """2^26 rows of 4096 sequences, all but four of them padding: as one dimension the merge would have 2^32 lanes."""
    b, t, g, d, cap = 4096, 128, 128, 64, 144
    assert b * t * g * 64 >= 1 << 32
    small = plain.Cache(2, 1, d, cap)
    small.fill([20, cap])
    at = torch.tensor([0, b - 1])                                      # the last sequence has two chunks
    planes = {}
    for w in "kv":
        planes[w + "c"] = torch.zeros(b, 1, cap, d // 2, dtype=torch.uint8, device="cuda")
        planes[w + "s"] = torch.zeros(b, 1, d // 32, cap, dtype=torch.float16, device="cuda")
        planes[w + "c"][at] = torch.from_numpy(small.codes[w]).cuda()
        planes[w + "s"][at] = torch.from_numpy(small.scales[w]).cuda()
    desc = rocm.Kv4Cache(*[planes[n].data_ptr() for n in ("kc", "ks", "vc", "vs")], None, b, 1, d, cap, 0, 0)
    lens, counts = torch.full((b,), cap, dtype=torch.int32), torch.zeros(b, dtype=torch.int32)
    lens[0], counts[at] = 20, 2
    lens, counts = lens.cuda(), counts.cuda()
    q = query(1, 2, 2, g, d)
    qd, out = torch.empty(b, t, g, d, device="cuda"), torch.full((b, t, g, d), POISON, device="cuda")
    qd[at, :2] = torch.from_numpy(q).cuda()
    torch.cuda.synchronize()
    rocm.call("aljabr_rocm_kv4_attention", out.data_ptr(), qd.data_ptr(), ctypes.byref(desc), lens.data_ptr(), counts.data_ptr(), t, g,
              0.0, 1, 0, 0.0, None, 0)
    torch.cuda.synchronize()
    check(out[at, :2].cpu().numpy(), *plain.attention(small, q, [20, cap]))
    assert (out[at, 2:] == POISON).all()
    assert all(bool((out[s:s + 128] == POISON).all()) for s in range(128, b - 128, 128))
    assert (out[1:128] == POISON).all() and (out[b - 128:b - 1] == POISON).all()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("t", [1, 6, 40])
@pytest.mark.parametrize("n", [200, 224])
@pytest.mark.parametrize("scale,most", [(8192.0, 7), (-12000.0, 5), (30000.0, 2), (65504.0, 1)])
def test_scales_past_the_writers_with_finite_values(rocm, d, t, n, scale, most):
    """Visible keys of another writer: a scale past 8160 whose codes keep every value within fp16, wherever tiles end."""
    host = plain.Cache(1, 2, d, 240)
    host.fill([n])
    q = query(d + n, 1, t, 8, d)
    rng = np.random.default_rng(most)
    for pos in (0, 31, 100, n - t, n - 5, n - 1):                      # of 40 rows, the last are seen by some only
        at = rng.integers(0, d // 32)                                  # one block
        c = rng.integers(8 - most, 9 + most, (2, 32)).astype(np.uint8)
        host.codes["v"][0, :, pos, 16 * at:16 * at + 16] = c[:, :16] | c[:, 16:] << 4
        host.scales["v"][0, :, at, pos] = scale
    want, bound, live = plain.attention(host, q, [n])
    assert np.isfinite(want).all()
    check(attend(rocm, Device(rocm, host), q, [n]), want, bound, live)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("t", [6, 40])
def test_values_past_fp16_reach_only_rows_that_see_them(rocm, d, t):
    """One value of a key that two rows see leaves fp16: those rows' block may be NaN, nothing else."""
    host = plain.Cache(1, 1, d, 128)
    host.fill([101])
    q = query(d + t, 1, t, 4, d)
    want, bound, live = plain.attention(host, q, [101])
    for block in range(d // 32):
        saved = [host.codes["v"].copy(), host.scales["v"].copy()]
        c = np.full(32, 9, np.uint8)
        c[(7 * block + 3) % 32] = 0                                    # -8 of a scale of 30000
        host.codes["v"][0, 0, 99, 16 * block:16 * block + 16] = c[:16] | c[16:] << 4
        host.scales["v"][0, 0, block, 99] = 30000.0
        got = attend(rocm, Device(rocm, host), q, [101])
        check(got[:, :t - 2], want[:, :t - 2], bound[:, :t - 2], live[:, :t - 2])
        other = [i for i in range(d) if i // 32 != block]
        assert (np.abs(got - want)[0, t - 2:][..., other] <= bound[0, t - 2:][..., other]).all()
        assert (~np.isfinite(got[0, t - 2:, :, 32 * block + (7 * block + 3) % 32])).all()
        host.codes["v"], host.scales["v"] = saved


@pytest.mark.parametrize("d,t", [(64, 1), (128, 5), (256, 1), (128, 40), (256, 40)])
@pytest.mark.parametrize("cap", [3.4e38, 1e38, 1e30, 2.0 ** 64, 1e10])
def test_soft_caps_past_every_score(rocm, d, t, cap):
    """cap tanh(score / cap) of a cap far past the scores is the score; the bound is that without a cap (its terms in cap are
    bounds for |score| near cap), and 4 roundings of each score for the cap's products and tanh."""
    host = plain.Cache(2, 1, d, 208)
    host.fill([200, 9])
    q = query(t, 2, t, 4, d)
    want, bound, live = plain.attention(host, q, [200, 9])
    k = host.rows_of("k", 0, 200)[0].astype(np.float64)
    top = (np.abs(k) @ np.abs(q[0].reshape(-1, d).T)).max() * d ** -0.5
    v = np.abs(host.rows_of("v", 0, 200)[0].astype(np.float64)).max()
    check(attend(rocm, Device(rocm, host), q, [200, 9], cap=cap), want, bound + 2 * v * 4 * top * 2.0 ** -24, live)


@pytest.mark.parametrize("d,t", [(64, 1), (128, 5), (256, 1), (128, 40), (256, 40)])
@pytest.mark.parametrize("cap,size", [(1e-6, 1.0), (1e-20, 1.0), (1e-38, 1.0), (1e-44, 1.0), (1e-6, 1e30), (1e-30, 1e25), (1e-44, 1e30)])
def test_soft_caps_next_to_zero(rocm, d, t, cap, size):
    """Scores of at most 1e-6: every key weighs the same to 2e-6. Keys of zeros, whose scores are 0, are among them."""
    host = plain.Cache(2, 1, d, 208)
    host.fill([200, 9])
    for pos in (0, 8):
        host.write("k", 1, pos, np.zeros((1, d), np.float32))
    q = query(t, 2, t, 4, d) * np.float32(size)
    want, bound, live = plain.attention(host, np.zeros_like(q), [200, 9])
    v = np.abs(host.rows_of("v", 0, 200)[0].astype(np.float64)).max()
    check(attend(rocm, Device(rocm, host), q, [200, 9], cap=cap), want, bound + 2 * 2 * 1e-6 * v, live)


@pytest.mark.parametrize("d,t", [(64, 1), (128, 5), (256, 1), (128, 40), (256, 40)])
@pytest.mark.parametrize("scale,size", [(3.4e38, 1e-39), (2.5e38, 1e-38), (1e-38, 2e37), (2e-39, 1e38), (1e30, 1e-31)])
def test_scales_at_the_ends_of_fp32(rocm, d, t, scale, size):
    host = plain.Cache(1, 1, d, 208)
    host.fill([200])
    with np.errstate(over="ignore"):
        q = query(t, 1, t, 4, d) * np.float32(size)
    scale = float(np.float32(scale))
    want, bound, live = plain.attention(host, q, [200], scale=scale)
    # Scores are far apart here: a weight's second fp16 part, of 2^13 times the weight or more, is off by up to 2^-25, so a
    # weight by up to 2^-38 of the largest, which a dim where the largest weight's value is 0 shows: 200 of them, on values
    # of at most v, over a sum of at least the largest.
    v = np.abs(host.rows_of("v", 0, 200)[0].astype(np.float64)).max()
    got = attend(rocm, Device(rocm, host), q, [200], scale=scale)
    past = ~np.isfinite(q).all(-1)                                     # at 1e38 some element is infinite: its row is NaN
    assert np.isnan(got[past]).all() and np.isnan(want[past]).all()
    got, want, bound = (np.where(past[..., None], 0.0, x) for x in (got, want, bound))
    check(got, want, bound + 200 * 2.0 ** -38 * v, live)


@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("t", [1, 6, 40])
def test_bad_blocks_at_other_head_sizes(rocm, d, t):
    lens = [90, 90, 90, 20]
    host = plain.Cache(4, 2, d, 96, 16)
    host.fill(lens)
    host.table[0, 2], host.table[1, 0], host.table[1, 5], host.table[3, :] = -1, host.s, 2 ** 31 - 1, -5
    q = query(6, 4, t, 8, d)
    got = attend(rocm, Device(rocm, host), q, lens)
    check(got, *plain.attention(host, q, lens))
    assert not got[3].any()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("t,window", [(4, 0), (40, 0), (4, 50), (40, 60)])
def test_nan_in_each_block_reaches_its_dims_of_the_rows_that_see_it(rocm, d, t, window):
    """V of one key the last two rows see, and of one that leaves the windows after the first: NaN in one block of 32 dims
    after the other, which those rows have there, and the others nowhere."""
    n = 100
    host = plain.Cache(1, 2, d, 128)
    host.fill([n])
    q = query(8, 1, t, 4, d)
    clean = plain.attention(host, q, [n], window=window)
    keys = [n - 2] + ([n - t - window + 1] if window else [])
    rng = np.random.default_rng(d)
    for block in range(d // 32):
        saved = [host.codes["v"].copy(), host.scales["v"].copy()]
        for key in keys:
            x = rng.standard_normal((2, d)).astype(np.float32)
            x[1, 32 * block + 5] = np.nan
            host.write("v", 0, key, x)
        want, bound, _ = plain.attention(host, q, [n], window=window)
        got = attend(rocm, Device(rocm, host), q, [n], window=window)
        hurt = np.zeros(got.shape, bool)
        hurt[0, t - 2:, 2:, 32 * block:32 * block + 32] = True
        if window:
            hurt[0, 0, 2:, 32 * block:32 * block + 32] = True
        assert np.array_equal(np.isnan(want), hurt) and np.array_equal(np.isnan(got), hurt)
        assert (np.abs(got - want)[~hurt] <= bound[~hurt]).all()
        host.codes["v"], host.scales["v"] = saved
    check(attend(rocm, Device(rocm, host), q, [n], window=window), *clean)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("t,g", [(1, 4), (5, 4), (40, 2)])
@pytest.mark.parametrize("scale", [1.0, 0.01])
def test_queries_and_weights_have_two_parts(rocm, d, t, g, scale):
    """Keys of one number each, for which the bound does not hold with one fp16 part (tests/test_kv4.py)."""
    host, q = plain.one_hot_keys(d), plain.one_hot_query(d, t, g)
    check(attend(rocm, Device(rocm, host), q, [40], scale=scale), *plain.attention(host, q, [40], scale=scale))
