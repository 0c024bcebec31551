"""fp16 and fp32 KV caches without a GPU: what the calls refuse, plane sizes, and
the plain forms that the GPU tests compare with."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

import kv_plain as plain
from aljabr_amd import abi

P = 0x10000                                                # a device pointer that no call gets to use


def cache(**kw):
    f = dict(k=P, v=0x20000, block_table=None, type=1, layers=2, sequences=2, n_kv_heads=8, head_dim=128, rows=64, num_blocks=0,
             max_blocks=0)
    f.update(kw)
    return abi.KvCache(*[f[n] for n, _ in abi.KvCache._fields_])


PAGED = dict(block_table=0x30000, num_blocks=16, max_blocks=4, rows=16)


def append(c, layer=0, q_out=0x100000, q=0x200000, k=0x300000, v=0x400000, pos=0x500000, t=1, hq=32, qs=(0, 0, 0), kvs=(0, 0, 0),
           type=0, rotation=abi.Rotation(1e4, 0, 0, None)):
    return abi.load().aljabr_rocm_kv_append(None if c is None else ctypes.byref(c), layer, q_out, q, k, v, pos, None, None, t, hq, *qs, *kvs,
                                            type, None if rotation is None else ctypes.byref(rotation))


def attend(c, layer=0, out=P, q=P, lens=P, parents=None, t=1, hq=32, scale=0.0, cap=0.0, ws=None):
    return abi.load().aljabr_rocm_kv_tree_attention(out, q, None if c is None else ctypes.byref(c), layer, lens, None, parents, t, hq, scale,
                                                    0, cap, ws, 0)


def accept(c, outs=(0x1000, 0x2000, 0x3000, 0x4000), lens=0x5000, counts=None, parents=0x6000, tokens=0x7000, choices=0x8000, t=8):
    return abi.load().aljabr_rocm_kv_tree_accept(None if c is None else ctypes.byref(c), *outs, lens, counts, parents, tokens, choices, t)


CALLS = [append, attend, accept]


@pytest.mark.parametrize("call", CALLS)
def test_without_init(call):
    lib = abi.load()
    if lib.aljabr_rocm_is_initialized():
        pytest.skip("the library is initialised")
    assert call(cache()) == -1
    assert call(cache(**PAGED)) == -1


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("bad", [dict(k=None), dict(v=None), dict(k=P + 8), dict(v=P + 4), dict(layers=0), dict(sequences=0),
                                 dict(sequences=-1), dict(n_kv_heads=0), dict(head_dim=0), dict(rows=0), dict(rows=-16),
                                 dict(rows=(1 << 30) + 1), dict(sequences=65536), dict(n_kv_heads=16385, rows=1),
                                 dict(num_blocks=4), dict(max_blocks=4), dict(num_blocks=-1), dict(PAGED, rows=24),
                                 dict(PAGED, num_blocks=0), dict(PAGED, max_blocks=0), dict(PAGED, max_blocks=-1),
                                 dict(PAGED, max_blocks=(1 << 26) + 1), dict(layers=1 << 30, sequences=65535, n_kv_heads=16384, rows=1 << 30)])
def test_bad_caches(call, bad):
    assert call(cache(**bad)) == -2


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("bad", [dict(head_dim=96), dict(head_dim=512), dict(type=2), dict(type=30)])
def test_caches_without_a_kernel(call, bad):
    assert call(cache(**bad)) == -3


@pytest.mark.parametrize("call", CALLS)
def test_no_cache(call):
    assert call(None) == -2


@pytest.mark.parametrize("layer", [-1, 2])
def test_layers_that_are_not_there(layer):
    assert append(cache(), layer=layer) == -2
    assert attend(cache(), layer=layer) == -2


@pytest.mark.parametrize("kw", [dict(q=None, q_out=None, k=None, v=None), dict(q=None), dict(q_out=None), dict(pos=None), dict(t=0),
                                dict(t=-1), dict(t=(1 << 30) + 1), dict(hq=0), dict(hq=65537), dict(qs=(-1, 1, 1)), dict(kvs=(1, 1, -1)),
                                dict(q=0x200002), dict(k=0x300001), dict(q_out=0x100008), dict(t=1 << 30),
                                dict(rotation=abi.Rotation(0.0, 0, 0, None)), dict(rotation=abi.Rotation(-1.0, 0, 0, None)),
                                dict(rotation=abi.Rotation(float("inf"), 0, 0, None)), dict(rotation=abi.Rotation(float("nan"), 0, 0, None)),
                                dict(rotation=abi.Rotation(1e4, 136, 0, None)), dict(rotation=abi.Rotation(1e4, -8, 0, None)),
                                dict(rotation=abi.Rotation(1e4, 0, 0, 0x2))])
def test_bad_appends(kw):
    assert append(cache(), **kw) == -2


@pytest.mark.parametrize("kw", [dict(type=1), dict(qs=(2 * 48 * 128, 48 * 128, 128)), dict(qs=(2 * 32 * 128, 128, 256)),
                                dict(qs=(4 * 32 * 128, 32 * 128, 128))])
def test_rows_in_place_are_dense_fp32(kw):
    """q_out as Q: any other row would be written over before it is read."""
    assert append(cache(), q_out=0x200000, t=2, **kw) == -2
    if not abi.load().aljabr_rocm_is_initialized():                       # else they would run, on no memory
        assert append(cache(), q_out=0x200000, t=2) == -1 == append(cache(), q_out=0x200000, t=2, qs=(2 * 32 * 128, 32 * 128, 128))


@pytest.mark.parametrize("kw", [dict(type=2), dict(type=-1), dict(rotation=abi.Rotation(1e4, 12, 0, None))])
def test_appends_without_a_kernel(kw):
    assert append(cache(), **kw) == -3


@pytest.mark.parametrize("kw", [dict(out=None), dict(q=None), dict(lens=None), dict(t=0), dict(hq=0), dict(hq=12), dict(out=P + 4),
                                dict(q=P + 8), dict(ws=P + 8), dict(scale=float("nan")), dict(cap=float("inf")), dict(t=1 << 26)])
def test_bad_attention(kw):
    assert attend(cache(), **kw) == -2


def test_sizes_that_attention_refuses():
    assert attend(cache(), t=257, parents=P) == -3
    big = dict(block_table=0x50000, num_blocks=1 << 20, rows=64, max_blocks=1 << 24)
    assert attend(cache(**dict(big, sequences=33))) == -2                 # 33 of 2^30 positions
    # The positions' tiles, of 16 keys for fp32, are added up in 32 bits: 2^31 of them would pass those.
    assert attend(cache(**dict(big, sequences=32, type=0))) == -2
    assert attend(cache(**dict(big, sequences=17))) == -2
    n = ctypes.c_size_t()
    assert abi.load().aljabr_rocm_kv_tree_attention_workspace(ctypes.byref(cache(**dict(big, sequences=16))), 1, 32, ctypes.byref(n)) in (0, -1)
    assert abi.load().aljabr_rocm_kv_tree_attention_workspace(ctypes.byref(cache()), 1, 12, ctypes.byref(n)) == -2
    assert abi.load().aljabr_rocm_kv_tree_attention_workspace(ctypes.byref(cache()), 1, 32, None) == -2


@pytest.mark.parametrize("kw", [dict(outs=(None, 0x2000, 0x3000, 0x4000)), dict(outs=(0x1000, None, 0x3000, 0x4000)),
                                dict(outs=(0x1000, 0x2000, None, 0x4000)), dict(outs=(0x1000, 0x2000, 0x3000, None)), dict(lens=None),
                                dict(tokens=None), dict(choices=None), dict(t=0), dict(t=-3), dict(lens=0x1000), dict(tokens=0x2000),
                                dict(choices=0x4000), dict(parents=0x2000), dict(counts=0x3000)])
def test_bad_accepts(kw):
    assert accept(cache(), **kw) == -2


def test_accept_of_more_rows_than_a_tree():
    assert accept(cache(), t=257) == -3


def test_cache_bytes():
    n, lib = ctypes.c_size_t(7), abi.load()
    ask = lambda **kw: lib.aljabr_rocm_kv_cache_bytes(ctypes.byref(cache(k=None, v=None, **kw)), ctypes.byref(n))
    assert ask() == 0 and n.value == 2 * 2 * 8 * 64 * 128 * 2
    assert ask(type=0, rows=33) == 0 and n.value == 2 * 2 * 8 * 33 * 128 * 4
    assert ask(num_blocks=10, rows=16) == 0 and n.value == 2 * 10 * 8 * 16 * 128 * 2
    assert ask(num_blocks=10, rows=16, sequences=0) == 0
    n.value = 7
    assert ask(sequences=0) == -2 and ask(head_dim=32) == -3 and ask(num_blocks=4, rows=20) == -2
    assert ask(num_blocks=1 << 30, layers=1 << 20, rows=1 << 20) == -2 and n.value == 7
    assert lib.aljabr_rocm_kv_cache_bytes(None, ctypes.byref(n)) == -2
    assert lib.aljabr_rocm_kv_cache_bytes(ctypes.byref(cache()), None) == -2


# ---- the plain forms -------------------------------------------------------------------

def test_a_chain_is_causal():
    host = plain.Cache(2, 2, 64, 40)
    host.fill([30, 17])
    q = np.random.default_rng(0).standard_normal((2, 5, 4, 64)).astype(np.float32)
    want = plain.attention(host, q, [30, 17], [5, 3])
    trees = np.stack([plain.chain(5)] * 2)
    got = plain.attention(host, q, [30, 17], [5, 3], trees)
    assert np.array_equal(want[0], got[0]) and np.array_equal(want[2], got[2])
    k, v = (host.rows_of(w, 0, 30)[0] for w in "kv")
    s = np.exp(q[0, 2, 1].astype(np.float64) @ k[0, :28].T / 8)
    assert np.allclose(got[0][0, 2, 1], s @ v[0, :28] / s.sum(), rtol=1e-12, atol=1e-12)


def test_accepting_rows_is_decoding_in_order():
    """The path's tokens are what the model chose one after the other, and its rows lie in order."""
    rng = np.random.default_rng(3)
    host = plain.Cache(4, 1, 64, 64, 16, layers=2)
    host.fill([40] * 4)
    parents = plain.random_parents(rng, 4, 20)
    tokens, choices = rng.integers(0, 3, (4, 20)), rng.integers(0, 3, (4, 20))
    before = [host.rows_of("k", b, 40, 1)[0] for b in range(4)]
    new_lens, path, accepted, after = plain.accept(host, [40] * 4, None, parents, tokens, choices)
    assert accepted.max() > 1
    for b in range(4):
        p = path[b, :accepted[b]]
        assert p[0] == 0 and (path[b, accepted[b]:] == -1).all() and new_lens[b] == 20 + accepted[b]
        assert all(parents[b, y] == x and tokens[b, y] == choices[b, x] for x, y in zip(p, p[1:]))
        assert after[b] == choices[b, p[-1]]
        assert np.array_equal(host.rows_of("k", b, new_lens[b], 1)[0][:, 20:], before[b][:, 20 + p])


@pytest.mark.parametrize("interleaved", [0, 1])
def test_rotation_keeps_distances(interleaved):
    """The product of a query and a key depends on the distance of their positions alone."""
    rng = np.random.default_rng(1)
    q, k = rng.standard_normal((2, 64))
    dot = lambda a, b: plain.rotate(q, a, 1e4, 48, interleaved, None)[0] @ plain.rotate(k, b, 1e4, 48, interleaved, None)[0]
    assert abs(dot(7, 3) - dot(1004, 1000)) < 1e-9
    assert np.array_equal(plain.rotate(q, 5, 1e4, 48, interleaved, None)[0][48:], q[48:])
