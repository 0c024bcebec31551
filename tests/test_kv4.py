"""The 4-bit KV cache without a GPU: sizes, refusals, and the plain encoder's own rules."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

import kv4_plain as plain
from aljabr_amd import abi


def cache(**kw):
    """A description of a cache whose planes are never touched."""
    base = dict(k_codes=0x10000, k_scales=0x20000, v_codes=0x30000, v_scales=0x40000, block_table=None, sequences=2,
                n_kv_heads=8, head_dim=128, rows=64, num_blocks=0, max_blocks=0)
    base.update(kw)
    return abi.Kv4Cache(*[base[n] for n, _ in abi.Kv4Cache._fields_])


def test_cache_bytes():
    lib = abi.load()
    codes, scales = ctypes.c_size_t(), ctypes.c_size_t()
    assert lib.aljabr_rocm_kv4_cache_bytes(ctypes.byref(cache()), ctypes.byref(codes), ctypes.byref(scales)) == 0
    assert (codes.value, scales.value) == (2 * 8 * 64 * 64, 2 * 8 * 64 * 4 * 2)
    big = cache(sequences=1, num_blocks=1 << 20, rows=128, head_dim=256)
    assert lib.aljabr_rocm_kv4_cache_bytes(ctypes.byref(big), ctypes.byref(codes), ctypes.byref(scales)) == 0
    assert codes.value == (1 << 20) * 8 * 128 * 128                      # past 32 bits
    for bad in (dict(rows=40), dict(rows=0), dict(n_kv_heads=0), dict(sequences=0)):
        assert lib.aljabr_rocm_kv4_cache_bytes(ctypes.byref(cache(**bad)), ctypes.byref(codes), ctypes.byref(scales)) == -2
    assert lib.aljabr_rocm_kv4_cache_bytes(ctypes.byref(cache(head_dim=96)), ctypes.byref(codes), ctypes.byref(scales)) == -3
    assert lib.aljabr_rocm_kv4_cache_bytes(None, ctypes.byref(codes), ctypes.byref(scales)) == -2


BAD_CACHES = [
    (dict(k_codes=None), -2), (dict(v_scales=None), -2), (dict(sequences=0), -2), (dict(sequences=70000), -2),
    (dict(n_kv_heads=-1), -2), (dict(rows=24), -2), (dict(rows=0), -2), (dict(k_codes=0x10008), -2), (dict(v_scales=0x40002), -2),
    (dict(block_table=0x50000), -2), (dict(block_table=0x50000, num_blocks=4), -2),
    (dict(block_table=0x50000, num_blocks=4, max_blocks=1 << 27), -2), (dict(head_dim=96), -3), (dict(head_dim=512), -3),
]
P = 0x60000


@pytest.mark.parametrize("bad,status", BAD_CACHES)
def test_bad_caches_are_refused_by_every_call(bad, status):
    lib, c = abi.load(), ctypes.byref(cache(**bad))
    n = ctypes.c_size_t()
    assert lib.aljabr_rocm_kv4_write(c, P, P, P, None, 1, 0, 0, 0, abi.TYPE_F32) == status
    assert lib.aljabr_rocm_kv4_read(P, P, c, P, None, 1, 0, 0, 0, abi.TYPE_F32) == status
    assert lib.aljabr_rocm_kv4_attention(P, P, c, P, None, 1, 32, 0.0, 1, 0, 0.0, None, 0) == status
    assert lib.aljabr_rocm_kv4_attention_workspace(c, 1, 32, ctypes.byref(n)) == status
    assert abi.last_error()


def test_bad_arguments_are_refused():
    lib, c = abi.load(), ctypes.byref(cache())
    write, read, att = lib.aljabr_rocm_kv4_write, lib.aljabr_rocm_kv4_read, lib.aljabr_rocm_kv4_attention
    for fn in (lambda k, v, pos, t, sb, st, sh, ty: write(c, k, v, pos, None, t, sb, st, sh, ty),
               lambda k, v, pos, t, sb, st, sh, ty: read(k, v, c, pos, None, t, sb, st, sh, ty)):
        assert fn(None, None, P, 1, 0, 0, 0, 0) == -2          # neither K nor V
        assert fn(P, P, None, 1, 0, 0, 0, 0) == -2
        assert fn(P, P, P, 0, 0, 0, 0, 0) == -2
        assert fn(P, P, P, -3, 0, 0, 0, 0) == -2
        assert fn(P, P, P, 1, 0, -128, 0, 0) == -2
        assert fn(P + 2, P, P, 1, 0, 0, 0, 0) == -2            # fp32 off its element
        assert fn(P, P, P, 1, 0, 0, 0, abi.TYPE_Q8_0) == -3
    bad = [dict(out=None), dict(q=None), dict(lens=None), dict(t=0), dict(hq=12), dict(hq=0), dict(out=P + 4), dict(q=P + 8),
           dict(ws=P + 4), dict(scale=float("nan")), dict(cap=float("inf"))]
    for b in bad:
        a = dict(out=P, q=P, lens=P, t=1, hq=32, scale=0.0, cap=0.0, ws=None)
        a.update(b)
        assert att(a["out"], a["q"], c, a["lens"], None, a["t"], a["hq"], a["scale"], 1, 0, a["cap"], a["ws"], 0) == -2, b
    assert lib.aljabr_rocm_kv4_attention_workspace(c, 1, 32, None) == -2


def test_encoder_rules():
    x = np.zeros((4, 64), np.float32)
    x[0, 3], x[0, 40] = -4.0, 4.0                              # the largest magnitude takes code 0 whatever its sign
    x[1, :32] = np.arange(32) - 16
    x[2, 5], x[2, 6] = 8.0, -8.0                               # two alike: the negative one
    x[3, 0] = np.inf
    codes, scales = plain.encode(x)
    v = plain.decode(codes, scales).astype(np.float64)
    assert v[0, 3] == -4.0 and v[0, 40] == 4.0 and scales[0, 0] == 0.5 and scales[0, 1] == -0.5
    assert np.array_equal(v[1, ::2], x[1, ::2]) and scales[1, 0] == 2.0
    assert scales[2, 0] == 1.0 and v[2, 6] == -8.0 and v[2, 5] == 7.0
    assert np.isnan(v[3, :32]).all() and not v[3, 32:].any()


def test_encoder_is_within_half_a_step():
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((64, 256)) * np.exp(rng.uniform(-20, 9, (64, 1)))).astype(np.float32)
    codes, scales = plain.encode(x)
    err = np.abs(plain.decode(codes, scales).astype(np.float64) - x).reshape(64, 8, 32)
    step = np.abs(scales.astype(np.float64))[..., None]
    # Half a step; a whole one and the scale's rounding (2^-9 of 8 steps) for a value as large as the top one, of the other sign.
    top = np.abs(x).reshape(64, 8, 32) > 7.5 * step * (1 - 2.0 ** -8)
    assert (err <= np.where(top, 1 + 2.0 ** -6, 0.5) * step + 2.0 ** -25 * 8).all()


def test_limits_of_sizes():
    lib, n = abi.load(), ctypes.c_size_t()
    ask = lambda c, t=1, hq=32: lib.aljabr_rocm_kv4_attention(P, P, ctypes.byref(c), P, None, t, hq, 0.0, 1, 0, 0.0, None, 0)
    paged = dict(block_table=0x50000, num_blocks=1 << 20)
    assert ask(cache(rows=(1 << 26) + 16)) == -2
    assert ask(cache(max_blocks=(1 << 24) + 1, **paged)) == -2                     # 2^30 positions and a block
    assert ask(cache(sequences=33, max_blocks=1 << 24, **paged)) == -2             # 33 of 2^30: past 2^35
    assert ask(cache(), t=1 << 26) == -2                                           # T * Hq
    assert lib.aljabr_rocm_kv4_write(ctypes.byref(cache(max_blocks=(1 << 24) + 1, **paged)), P, P, P, None, 1, 0, 0, 0, 0) == -2
    assert "2^30" in abi.last_error()


@pytest.mark.parametrize("blocks", [dict(num_blocks=4), dict(max_blocks=4), dict(num_blocks=1, max_blocks=2), dict(num_blocks=-1)])
def test_blocks_without_a_table_are_refused(blocks):
    """kv4_cache_bytes sizes such planes by num_blocks: taken as contiguous, `sequences` may reach past them."""
    lib, c = abi.load(), ctypes.byref(cache(**blocks))
    n = ctypes.c_size_t()
    assert lib.aljabr_rocm_kv4_write(c, P, P, P, None, 1, 0, 0, 0, abi.TYPE_F32) == -2
    assert lib.aljabr_rocm_kv4_read(P, P, c, P, None, 1, 0, 0, 0, abi.TYPE_F32) == -2
    assert lib.aljabr_rocm_kv4_attention(P, P, c, P, None, 1, 32, 0.0, 1, 0, 0.0, None, 0) == -2
    assert lib.aljabr_rocm_kv4_attention_workspace(c, 1, 32, ctypes.byref(n)) == -2
    assert "block_table" in abi.last_error()


def test_cache_bytes_past_64_bits_are_refused():
    lib, codes, scales = abi.load(), ctypes.c_size_t(7), ctypes.c_size_t(7)
    ask = lambda **kw: lib.aljabr_rocm_kv4_cache_bytes(ctypes.byref(cache(**kw)), ctypes.byref(codes), ctypes.byref(scales))
    top = 2 ** 31 - 1
    assert ask(num_blocks=top, n_kv_heads=top, rows=top - 15, head_dim=256) == -2
    assert ask(num_blocks=1 << 30, n_kv_heads=1 << 14, rows=1 << 20, head_dim=64) == -2     # 2^69: 0 in 64 bits
    assert ask(sequences=1 << 29, n_kv_heads=1 << 15, rows=1 << 15, head_dim=64) == -2      # codes 2^64
    assert (codes.value, scales.value) == (7, 7)
    assert ask(sequences=1 << 28, n_kv_heads=1 << 15, rows=1 << 15, head_dim=64) == 0       # codes 2^63
    assert (codes.value, scales.value) == (1 << 63, 1 << 60)


@pytest.mark.parametrize("d,t", [(64, 1 << 29), (128, 1 << 28), (256, 1 << 27), (256, 1 << 30)])
def test_rows_of_more_than_one_launch_are_refused(d, t):
    """T rows of D / 8 lanes each: a launch takes fewer than 2^32."""
    lib, c = abi.load(), ctypes.byref(cache(head_dim=d))
    assert lib.aljabr_rocm_kv4_write(c, P, P, P, None, t, 0, 0, 0, abi.TYPE_F32) == -2
    assert "launch" in abi.last_error()
    assert lib.aljabr_rocm_kv4_read(P, P, c, P, None, t, 0, 0, 0, abi.TYPE_F16) == -2


@pytest.mark.parametrize("strides,shape", [((0, 128, 256), (2, 5, 2)), ((4096, 0, 128), (2, 5, 2)), ((4096, 128, 0), (2, 5, 2)),
                                           ((4096, 128, 0), (1, 1, 2))])
def test_read_into_rows_on_one_place_is_refused(strides, shape):
    """A stride of 0 reads a shared source row for several heads, tokens or sequences; what is read back has no such place."""
    lib = abi.load()
    b, t, h = shape
    c = ctypes.byref(cache(sequences=b, n_kv_heads=h))
    assert lib.aljabr_rocm_kv4_read(P, P, c, P, None, t, *strides, abi.TYPE_F32) == -2
    assert "stride" in abi.last_error()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("t,g", [(1, 4), (5, 4), (40, 2)])
def test_the_bound_tells_two_parts_from_one(d, t, g):
    """With keys of one number each the bound of kv4_plain.attention holds for queries and weights in two fp16 parts, with
    most of it to spare, and not for either in one."""
    host, q = plain.one_hot_keys(d), plain.one_hot_query(d, t, g)
    over = lambda scale, *parts: (np.abs(plain.in_fp16_parts(host, q, 40, scale, *parts) - want[scale][0]) / (want[scale][1] + 1e-30)).max()
    want = {scale: plain.attention(host, q, [40], scale=scale) for scale in (1.0, 0.01)}
    assert over(1.0, 2, 2) < 0.1 and over(0.01, 2, 2) < 0.1
    assert over(1.0, 1, 2) > 2                                 # queries in one part: scores of some size
    assert over(0.01, 2, 1) > 4                                # weights in one part: scores next to 0
