"""fp16 and fp32 KV caches at their ends and limits: drafts that reach past the
last place, numbers at the ends of their types."""
from __future__ import annotations

import copy
import ctypes

import numpy as np
import pytest
import torch

import kv_plain as plain
from test_gpu_kv_cache import F16, F32, POISON, ROOM, Device, agreeing, append, attend, check, check_planes, ints, normal, ptr, take

pytestmark = pytest.mark.gpu


# ---- drafts that reach past the end of the cache ----------------------------------------

def unending(host):
    """The host's cache as one that goes on past its end, where it has no rows: what lengths say is then not cut."""
    far = copy.copy(host)
    far.cap = 1 << 30
    far.at = host.at
    return far


def overhanging(cap, t):
    """Lengths and counts of four sequences: three rows in the cache, one, none, and none with a gap before them."""
    return [cap - 3 + t, cap - 1 + t, cap + t, cap + 9 + t], [t, t, t, max(t - 1, 1)]


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("cap,page", [(32, 16), (37, 0), (144, 48), (129, 0)])
@pytest.mark.parametrize("t,g", [(1, 4), (5, 2), (12, 4), (40, 3)])
@pytest.mark.parametrize("window", [0, 4, 30])
@pytest.mark.parametrize("tree", [0, 1])
def test_attention_of_drafts_past_the_end(rocm, d, dtype, cap, page, t, g, window, tree):
    host = plain.Cache(4, 2, d, cap, page, dtype)
    host.fill([cap] * 4)
    lens, counts = overhanging(cap, t)
    parents = plain.random_parents(np.random.default_rng(t), 4, t, window == 30) if tree else None
    q = normal(t, 4, t, 2 * g, d)
    got = attend(rocm, Device(rocm, host), q, lens, counts, parents, window)
    check(got, *plain.attention(unending(host), q, lens, counts, parents, window))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [0, 64])
@pytest.mark.parametrize("window", [0, 16470])
@pytest.mark.parametrize("tree", [0, 1])
def test_attention_of_many_rows_past_the_end(rocm, d, page, window, tree):
    """As above for the kernel that many rows over a large cache take."""
    t, cap = 33, 16512
    host = plain.Cache(2, 4, d, cap, page, F16)
    host.fill([cap] * 2)
    parents = plain.random_parents(np.random.default_rng(d), 2, t, True) if tree else None
    q = normal(d, 2, t, 16, d)
    for lens, counts in (([cap - 3 + t, cap - 20 + t], [t, t]), ([cap + t, cap + 9 + t], [t, t - 1])):
        got = attend(rocm, Device(rocm, host), q, lens, counts, parents, window)
        check(got, *plain.attention(unending(host), q, lens, counts, parents, window))


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("t,tree", [(1, 0), (7, 0), (7, 1), (40, 1)])
def test_lengths_far_past_the_end(rocm, dtype, t, tree):
    """At the largest length every row sees the whole cache, or none of it through a window."""
    host = plain.Cache(2, 2, 128, 70, 0, dtype)
    host.fill([70, 70])
    parents = plain.random_parents(np.random.default_rng(1), 2, t) if tree else None
    q, lens = normal(t, 2, t, 8, 128), [2 ** 31 - 1, 2 ** 31 - 1]
    dev = Device(rocm, host)
    check(attend(rocm, dev, q, lens, None, parents), *plain.attention(unending(host), q, [1000] * 2, None, parents))
    assert not attend(rocm, dev, q, lens, None, parents, 2 ** 30).any()
    assert not attend(rocm, dev, q, lens, None, parents, 5).any()
    assert np.array_equal(attend(rocm, dev, q, lens, None, parents, 2 ** 31 - 1), attend(rocm, dev, q, lens, None, parents))


@pytest.mark.parametrize("page", [0, 16])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_accept_at_the_end_of_the_cache(rocm, page, dtype):
    """29 committed rows of 32 and a draft of 5: row 2 is moved to the second place of the draft, no committed row changes."""
    host = plain.Cache(1, 2, 64, 32, page, dtype, 3)
    host.fill([32])
    before = [host.rows_of(w, 0, 32, layer)[0] for w in "kv" for layer in range(3)]
    dev = Device(rocm, host)
    got = take(rocm, dev, [34], None, np.array([[-1, 0, 0, 1, 2]]), np.array([[9, 1, 2, 3, 4]]), np.array([[2, 0, 8, 0, 0]]))
    assert [x.tolist() for x in got] == [[31], [[0, 2, -1, -1, -1]], [2], [8]]
    host.planes = {w: dev.plane(w) for w in "kv"}
    after = [host.rows_of(w, 0, 32, layer)[0] for w in "kv" for layer in range(3)]
    for x, y in zip(before, after):
        assert np.array_equal(x[:, :30], y[:, :30]) and np.array_equal(x[:, 31:], y[:, 31:])
        assert np.array_equal(y[:, 30], x[:, 31])


@pytest.mark.parametrize("d,dtype", [(64, F16), (128, F32), (256, F16)])
@pytest.mark.parametrize("t,cap,page", [(5, 32, 16), (5, 33, 0), (33, 48, 16), (64, 100, 0), (256, 300, 0)])
@pytest.mark.parametrize("deep", [0, 1])
def test_accept_of_drafts_past_the_end(rocm, d, dtype, t, cap, page, deep):
    rng = np.random.default_rng(t + d)
    parents = plain.random_parents(rng, 6, t, bool(deep))
    tokens, choices = agreeing(rng, parents, t, 0.97 if deep else 0.8, 4 if t < 9 else 50)
    lens, counts = [*overhanging(cap, t)[0], cap + t // 2, 2 ** 31 - 1], [*overhanging(cap, t)[1], t, t]
    host = plain.Cache(6, 3, d, cap, page, dtype, 2)
    host.fill([host.cap] * 6)
    dev = Device(rocm, host)
    got = take(rocm, dev, lens, counts, parents, tokens, choices)
    far = unending(host)
    far.cap = 1 << 40
    want = plain.accept(far, lens, counts, parents, tokens, choices)
    for x, y in zip(got, want):
        assert np.array_equal(x, y)
    check_planes(dev)


@pytest.mark.parametrize("page", [0, 16])
def test_a_step_at_the_end_of_the_cache(rocm, page):
    """Append, attention and accept of one draft that reaches past the end: they mean the same places."""
    b, t, d, cap = 3, 12, 64, 64
    rng = np.random.default_rng(page)
    host = plain.Cache(b, 2, d, cap, page, F16)
    base = [cap - 7, cap - 1, cap]
    host.fill(base)
    dev = Device(rocm, host)
    parents = plain.random_parents(rng, b, t, True)
    angles = np.array([[base[s] + len(plain.line(parents[s], i)) - 1 for i in range(t)] for s in range(b)])
    q, k, v = normal(1, b, t, 8, d), normal(2, b, t, 2, d), normal(3, b, t, 2, d)
    qd = append(rocm, dev, q, k, v, base, None, angles)
    turned, off, live, k_bound = plain.append(host, q, k, v, base, None, angles)
    assert (np.abs(qd - turned) <= off + 1e-30).all()
    check_planes(dev, k_bound)
    host.planes = {w: dev.plane(w) for w in "kv"}                      # from here on what the GPU's cache holds
    lens = [x + t for x in base]
    check(attend(rocm, dev, qd, lens, None, parents), *plain.attention(unending(host), qd, lens, None, parents))
    tokens, choices = agreeing(rng, parents, t, 0.95)
    got = take(rocm, dev, lens, None, parents, tokens, choices)
    want = plain.accept(unending(host), lens, None, parents, tokens, choices)
    for x, y in zip(got, want):
        assert np.array_equal(x, y)
    check_planes(dev)


# ---- numbers at the ends of their types -------------------------------------------------

@pytest.mark.parametrize("room", [0, ROOM])
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("d,t,tree", [(64, 1, 0), (128, 5, 0), (128, 12, 1), (256, 1, 0), (64, 40, 1), (128, 40, 0), (256, 40, 1)])
@pytest.mark.parametrize("scale,size", [(1e-38, 1e-3), (1e-44, 1.0), (1e-30, 1e-20), (1e-38, 1e-38), (1e-44, 3e38), (2e-20, 1e-30)])
def test_small_scales_of_small_queries(rocm, room, dtype, d, t, tree, scale, size):
    """Scores next to zero weigh all keys alike, and what a row does not see nothing."""
    host = plain.Cache(2, 1, d, 208, 0, dtype)
    host.fill([200, 77])
    q = np.float32(size) * np.clip(normal(t, 2, t, 4, d), -1, 1)
    parents = plain.random_parents(np.random.default_rng(t), 2, t) if tree else None
    scale = float(np.float32(scale))
    got = attend(rocm, Device(rocm, host, room), q, [200, 77], None, parents, scale=scale)
    check(got, *plain.attention(host, q, [200, 77], None, parents, scale=scale))


@pytest.mark.parametrize("room", [0, ROOM])
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("t,at", [(1, 40), (12, 40), (40, 40), (40, 95)])
@pytest.mark.parametrize("less", [10, 30, 60])
@pytest.mark.parametrize("seed", [1, 1000])
def test_infinite_values_of_small_weights(rocm, room, dtype, d, t, at, less, seed):
    """A value of a key whose score is far below the row's largest, `less` powers of e and more: its weight is not zero, and
    an infinity times it stays one, unless the weight is below fp32's range (2^-126 of the row's largest; seed 1 draws the
    queries like the keys, whose scores then reach 30)."""
    n = 100
    host = plain.Cache(1, 1, d, 128, 0, dtype)
    host.fill([n])
    host.planes["k"][0, 0, 0, :n, 7] = 0
    host.planes["k"][0, 0, 0, at, :] = 0
    host.planes["k"][0, 0, 0, at, 7] = -less
    host.planes["v"][0, 0, 0, at, 33] = np.inf
    host.planes["v"][0, 0, 0, at, 34] = -np.inf
    q = 0.1 * normal(seed, 1, t, 4, d)
    q[..., 7] = 1
    want, bound, live = plain.attention(host, q, [n], scale=1.0)
    got = attend(rocm, Device(rocm, host, room), q, [n], scale=1.0)
    fine = np.isfinite(want)
    assert (~fine).sum() == 2 * 4 * min(t, n - at)
    s = q[0].astype(np.float64) @ host.planes["k"][0, 0, 0, :n].astype(np.float64).T
    seen = np.arange(n) <= np.arange(n - t, n)[:, None]
    sure = (s[..., at] - np.where(seen[:, None], s, -np.inf).max(-1)) / np.log(2) > -126
    ends = ~fine & sure[None, ..., None]
    assert ends.any() and (ends.sum() == (~fine).sum() or less == 60)
    assert np.array_equal(got[ends], want[ends].astype(np.float32))
    rest = ~fine & ~ends
    assert (np.isnan(got[rest]) | (got[rest] == want[rest])).all()
    assert (np.abs(got[fine] - want[fine]) <= bound[fine]).all()


# ---- workspaces -------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("heads,t,g,d,cap", [(8, 5, 4, 128, 131072), (2, 8, 4, 64, 1 << 19), (8, 16, 4, 128, 65536), (4, 16, 8, 128, 65536),
                                             (8, 6, 4, 256, 65536)])
def test_the_advertised_workspace_is_enough_for_every_window(rocm, dtype, heads, t, g, d, cap):
    """A window may change how a call's work is laid out: with the advertised bytes it is cut as with any larger workspace."""
    page, blocks = 128, 64
    gen = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn(blocks, heads, page, d, device="cuda", generator=gen).to([torch.float32, torch.float16][dtype]) for _ in "kv")
    table = (torch.arange(cap // page, device="cuda", dtype=torch.int32) * 7 % blocks)[None].contiguous()
    desc = rocm.KvCache(k.data_ptr(), v.data_ptr(), table.data_ptr(), dtype, 1, 1, heads, d, page, blocks, cap // page)
    n = ctypes.c_size_t()
    rocm.call("aljabr_rocm_kv_tree_attention_workspace", ctypes.byref(desc), t, heads * g, ctypes.byref(n))
    assert n.value > 0
    q, lens = torch.randn(1, t, heads * g, d, device="cuda", generator=gen), ints([cap - 5])
    large = torch.zeros(2 * n.value + (1 << 20), dtype=torch.uint8, device="cuda")
    outs = [torch.empty_like(q) for _ in "ab"]
    for window in (0, cap - 1, cap // 2, cap // 4, 20000, 5000, 300, 20):
        for out, size in zip(outs, (n.value, large.numel())):
            torch.cuda.synchronize()
            rocm.call("aljabr_rocm_kv_tree_attention", out.data_ptr(), q.data_ptr(), ctypes.byref(desc), 0, lens.data_ptr(), None, None, t,
                      heads * g, 0.0, window, 0.0, large.data_ptr(), size)
        torch.cuda.synchronize()
        assert torch.equal(*outs), window


# ---- long chunks ----------------------------------------------------------------------------

@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("page", [0, 16, 112])
@pytest.mark.parametrize("t,g,room", [(1, 4, 0), (9, 2, 0), (20, 4, ROOM)])
@pytest.mark.parametrize("odd", [0, 1])
def test_one_chunk_of_many_keys(rocm, d, dtype, page, t, g, room, odd):
    """A workspace too small to cut the keys: each workgroup walks through all of them, further than the addresses that
    its lanes hold at once (the keys of 32 tiles a wave, or of 32 in all for many rows), blocks in any order, some of them
    not there; odd: with values that are not finite, for which it walks them again."""
    lens = [9841, 4300]
    host = plain.Cache(2, 1, d, 9850, page, dtype)
    host.fill(lens)
    if page:
        host.table[0, [2, 9000 // page]] = -1, host.s
        host.table[1, 3000 // page] = -7
    if odd:
        host.write("v", 0, 7003, np.where(np.arange(d) == 5, np.inf, 1.0)[None])
        host.write("v", 1, 4177, np.where(np.arange(d) == 50, np.nan, 1.0)[None])
        host.write("k", 1, 4100, np.where(np.arange(d) == 3, -np.inf, 0.0)[None])
    q = normal(t, 2, t, g, d)
    q[1, ..., 3] = np.abs(q[1, ..., 3])
    parents = plain.random_parents(np.random.default_rng(d), 2, t) if t > 1 else None
    want, bound, live = plain.attention(host, q, lens, None, parents)
    got = attend(rocm, Device(rocm, host, room), q, lens, None, parents, workspace=torch.zeros(16, dtype=torch.uint8, device="cuda"))
    fine = np.isfinite(want)
    assert (~fine).sum() == (2 * t * g if odd else 0)
    assert np.array_equal(got[~fine], want[~fine].astype(np.float32), equal_nan=True)
    check(np.where(fine, got, 0), np.where(fine, want, 0), np.where(fine, bound, 0), live)
