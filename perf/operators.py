"""The operators of a KV cache held in 4 bits, as this framework's speed in them
is measured: rows written, rows read back, and attention over the cache.

A row of head_dim values is held as blocks of 32 codes of 4 bits with one fp16
scale each, value = (code - 8) * scale. K and V each have two planes

    codes   uint8   [S][heads][R][head_dim / 2]    byte j of a block: code j | code (j + 16) << 4
    scales  float16 [S][heads][head_dim / 32][R]

with S sequences of R rows (contiguous), or S blocks of R = block rows that a
table hands to sequences (paged).

``own`` False computes every case in elementary torch operations over the same
planes; ``own`` True makes the calls of the framework's C ABI, as a serving
program does: one stream, stream-ordered calls, buffers allocated beforehand.
"""
from __future__ import annotations

import ctypes
import math

import torch

own = False

DEV = "cuda:0"
BLOCK = 32


# ---- the cases --------------------------------------------------------------------

def listed():
    return [
        # One token's K and V of a Llama-3-8B layer appended at batch 1, and read back: launches are all there is.
        dict(name="write_token_b1", kind="write", b=1, t=1, hkv=8, d=128, cap=2064, page=0, src="f32", rows="dense", ragged=0),
        # 64 sequences decoded together append to a paged cache, each at its own position.
        dict(name="write_token_b64_paged", kind="write", b=64, t=1, hkv=8, d=128, cap=2064, page=32, src="f32", rows="dense",
             ragged=0),
        # A prompt's K and V, slices of the stacked Q/K/V product's rows, four prompts of up to 2048 tokens.
        dict(name="write_prompt_b4_2048", kind="write", b=4, t=2048, hkv=8, d=128, cap=4096, page=0, src="f32", rows="qkv",
             ragged=1),
        # A short prefix of odd length handed back as fp16 rows per head, head size 64.
        dict(name="read_prefix_777_d64", kind="read", b=2, t=777, hkv=8, d=64, cap=1024, page=16, dst="f16", rows="heads", ragged=0),
        # Whole caches of 16 sequences turned back into the fp16 layout that the session's attention takes.
        dict(name="read_b16_8192", kind="read", b=16, t=8192, hkv=8, d=128, cap=8192, page=0, dst="f16", rows="heads", ragged=0),
        # Decode attention at batch 1, short context: latency.
        dict(name="decode_b1_512", kind="attention", b=1, t=1, hq=32, hkv=8, d=128, ctx=512, cap=2064, page=0, ragged=0,
             window=0, softcap=0.0),
        # Decode attention of 16 sequences at 4096 cached keys: the benchmark's attention shape.
        dict(name="decode_b16_4096", kind="attention", b=16, t=1, hq=32, hkv=8, d=128, ctx=4096, cap=4096, page=0, ragged=0,
             window=0, softcap=0.0),
        # A serving batch: 32 sequences of every length up to 4096 in pages of 16.
        dict(name="decode_b32_ragged_paged", kind="attention", b=32, t=1, hq=32, hkv=8, d=128, ctx=4096, cap=4096, page=16,
             ragged=1, window=0, softcap=0.0),
        # One very long context.
        dict(name="decode_b1_131072", kind="attention", b=1, t=1, hq=32, hkv=8, d=128, ctx=131072, cap=131072, page=0, ragged=0,
             window=0, softcap=0.0),
        # Drafts of up to five tokens verified, heads of 256 with a sliding window and a soft cap.
        dict(name="verify5_b8_window_d256", kind="attention", b=8, t=5, hq=16, hkv=8, d=256, ctx=4096, cap=4112, page=64,
             ragged=1, window=1024, softcap=50.0),
        # A 256-token chunk of a prompt against the earlier chunks.
        dict(name="chunk256_2048", kind="attention", b=1, t=256, hq=32, hkv=8, d=128, ctx=2048, cap=4096, page=0, ragged=0,
             window=0, softcap=0.0),
        # A whole prompt over the cache it has just been written to.
        dict(name="prompt2048", kind="attention", b=1, t=2048, hq=32, hkv=8, d=128, ctx=2048, cap=4096, page=0, ragged=0,
             window=0, softcap=0.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _rows16(n):
    return -(-n // 16) * 16


def draw(rng):
    """Another case of the listed ranges: any batch up to 64, rows from one
    token to whole prompts, contexts from one key to 131072, heads of 64, 128
    and 256 in any grouping, contiguous caches and pages of 16 to 128 rows."""
    kind = rng.choice(["write", "write", "read", "attention", "attention", "attention", "attention"])
    d = rng.choice([64, 128, 128, 256])
    page = rng.choice([0, 0, 16, 32, 64, 128])
    if kind in ("write", "read"):
        most = 8192 if kind == "write" else 65536
        b = rng.choice([1, _log(rng, 2, 64)])
        t = 1 if rng.random() < 0.3 else _log(rng, 2, most // b)
        hkv = rng.choice([1, 2, 4, 8, 8]) if d < 256 else rng.choice([1, 2, 4])
        cap = _rows16(t + rng.choice([0, 15, 100]))
        out = dict(kind=kind, b=b, t=t, hkv=hkv, d=d, cap=cap, page=page)
        if kind == "write":
            return dict(out, src=rng.choice(["f32", "f32", "f16"]), rows=rng.choice(["dense", "qkv", "heads"]),
                        ragged=rng.choice([0, 1]))
        return dict(out, dst=rng.choice(["f32", "f16", "f16"]), rows=rng.choice(["dense", "heads"]), ragged=rng.choice([0, 1]))
    hkv, g = rng.choice([(8, 4), (8, 4), (8, 8), (4, 8), (8, 1), (16, 2), (4, 7), (2, 3), (1, 16), (2, 12)])
    window, cap50 = rng.choice([(0, 0.0), (0, 0.0), (0, 0.0), (_log(rng, 16, 2048), 0.0), (1024, 50.0)])
    form = rng.choice(["decode", "decode", "verify", "chunk", "prompt"])
    if form in ("decode", "verify"):
        keys = (1 << 27) // (hkv * d)
        ctx = min(keys, _log(rng, 1 if form == "decode" else 16, 131072))
        b = max(1, min(_log(rng, 1, 64), keys // ctx))
        t = 1 if form == "decode" else rng.randint(2, 8)
    else:
        t = _log(rng, 9, 1024)
        b = 1 if t > 256 else rng.choice([1, 2, 4])
        ctx = t if form == "prompt" else min(t + _log(rng, 1, 4096), 4096)
        t = max(1, min(t, (1 << 34) // (b * ctx * hkv * g * d)))
        ctx = t if form == "prompt" else ctx
    return dict(kind=kind, b=b, t=t, hq=hkv * g, hkv=hkv, d=d, ctx=ctx, cap=_rows16(ctx + rng.choice([0, 15, 100])), page=page,
                ragged=rng.choice([0, 1]), window=window, softcap=cap50)


# ---- the format in plain torch ------------------------------------------------------

def _scale_and_codes(x):
    """[..., d] -> scales float32 [..., d / 32] and codes - 8 as float32 [..., d / 32, 32]."""
    x = x.float().reshape(*x.shape[:-1], -1, BLOCK)
    lo, hi = x.amin(-1), x.amax(-1)
    top = torch.where(-lo >= hi, lo, hi)
    step = top.abs() / 8
    # 8 significant bits, in steps of 2^-24 at the least: (code - 8) * scale is an fp16 number.
    step = torch.where(step >= 2.0 ** -17, step.bfloat16().float(), torch.round(step * 2.0 ** 24) * 2.0 ** -24)
    step = step.clamp(max=8160.0)
    scale = torch.where(top > 0, -step, step)
    # The quotient decides between codes: in float64 it lands on the right side of every border.
    q = torch.floor(x.double() / scale.double()[..., None] + 0.5).clamp_(-8, 7)
    q = torch.where(scale[..., None] == 0, torch.zeros_like(q), q).float()
    return scale, q


def _pack(q):
    """codes - 8 [..., d / 32, 32] -> bytes [..., d / 2]."""
    c = (q + 8).to(torch.uint8)
    return (c[..., :16] | (c[..., 16:] << 4)).flatten(-2)


def _unpack(codes, scales):
    """bytes [..., d / 2] and scales [..., d / 32] -> float32 values [..., d]."""
    c = codes.reshape(*codes.shape[:-1], -1, 16)
    q = torch.cat([c & 15, c >> 4], -1).float() - 8
    return (q * scales.float()[..., None]).flatten(-2)


def _row_index(table, pos, page):
    """The (sequence or block, row) of positions pos [b, t]."""
    if table is None:
        return torch.arange(pos.shape[0], device=pos.device)[:, None].expand_as(pos), pos
    return torch.gather(table.long(), 1, pos // page), pos % page


def _gather(state, which, s, r):
    """Rows (s, r) [b, t] of the K or V planes as float32 [b, t, heads, d]."""
    return _unpack(state[which + "_codes"][s, :, r], state[which + "_scales"][s, :, :, r])


# ---- what a program has in hand before the call --------------------------------------

class _Draw:
    """Seeded tensors on the device."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV).manual_seed(int(seed))

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.g, device=DEV)

    def ints(self, lo, hi, n):
        return torch.randint(lo, hi + 1, (n,), generator=self.g, device=DEV, dtype=torch.int32)


def _pair(g, b, t, hkv, d):
    """K and V rows [b, t, heads, d]: keys with the uneven channels that they have."""
    k = g.normal(b, t, hkv, d) * torch.exp(0.5 * g.normal(hkv, d))
    return k, g.normal(b, t, hkv, d)


def _planes(case, g, lens):
    """Empty planes of the case's cache and its table: blocks in shuffled order, -1 past a sequence's last."""
    b, hkv, d, cap, page = (case[n] for n in ("b", "hkv", "d", "cap", "page"))
    if page:
        per = -(-cap // page)
        s, r = b * per + 3, page
        table = torch.randperm(s, generator=g.g, device=DEV)[:b * per].int().reshape(b, per)
        used = (lens.long() + page - 1) // page
        table = torch.where(torch.arange(per, device=DEV)[None] < used[:, None], table, -1).int().contiguous()
    else:
        s, r, table = b, cap, None
    state = {"table": table}
    for which in "kv":
        state[which + "_codes"] = torch.zeros(s, hkv, r, d // 2, dtype=torch.uint8, device=DEV)
        state[which + "_scales"] = torch.zeros(s, hkv, d // BLOCK, r, dtype=torch.float16, device=DEV)
    return state


def _fill(case, state, g, lens):
    """Writes lens[b] rows of every sequence."""
    n = int(lens.max())
    step = max(1, (1 << 26) // (case["b"] * case["hkv"] * case["d"]))
    for t0 in range(0, n, step):
        t = min(step, n - t0)
        rows = _pair(g, case["b"], t, case["hkv"], case["d"])
        pos = torch.arange(t0, t0 + t, device=DEV)[None].expand(case["b"], t)
        keep = pos < lens.long()[:, None]
        at = torch.where(keep, pos, 0)
        s, r = _row_index(state["table"], at, case["page"])
        for which, x in zip("kv", rows):
            scale, q = _scale_and_codes(x)
            state[which + "_codes"][s[keep], :, r[keep]] = _pack(q)[keep]
            state[which + "_scales"][s[keep], :, :, r[keep]] = scale.half()[keep]


def _source(case, g):
    """K and V rows to be written and their strides (sequence, token, head), as the program holds them."""
    b, t, hkv, d = (case[n] for n in ("b", "t", "hkv", "d"))
    k, v = _pair(g, b, t, hkv, d)
    if case["src"] == "f16":
        k, v = k.half(), v.half()
    if case["rows"] == "dense":
        return (k, v), (k, v), (t * hkv * d, hkv * d, d)
    if case["rows"] == "heads":
        k, v = (x.transpose(1, 2).contiguous() for x in (k, v))
        return (k.transpose(1, 2), v.transpose(1, 2)), (k, v), (hkv * t * d, d, t * d)
    # Rows of a stacked Q/K/V product with four query heads a K/V head.
    row = 6 * hkv * d
    x = torch.zeros(b, t, row, dtype=k.dtype, device=DEV)
    views = tuple(x[:, :, o * hkv * d:(o + 1) * hkv * d].unflatten(-1, (hkv, d)) for o in (4, 5))
    for dst, src in zip(views, (k, v)):
        dst.copy_(src)
    return views, views, (t * row, row, d)


def _inputs(case, seed):
    """Everything of a case that the seed decides."""
    g, b, t = _Draw(seed), case["b"], case["t"]
    if case["kind"] == "attention":
        lens = g.ints(1, case["ctx"], b) if case["ragged"] else torch.full((b,), case["ctx"], dtype=torch.int32, device=DEV)
        lens[0] = case["ctx"]
        # A draft or chunk is padded to t rows: the last `counts` keys belong to its rows.
        counts = torch.minimum(g.ints(1, t, b), lens) if case["ragged"] and t > 1 else None
        state = _planes(case, g, lens)
        _fill(case, state, g, lens)
        return dict(state, lens=lens, counts=counts, q=g.normal(b, t, case["hq"], case["d"]))
    start = g.ints(0, case["cap"] - t, b)
    counts = g.ints(0, t, b) if case["ragged"] else None
    if counts is not None:
        counts[0] = t
    state = _planes(case, g, start + t)
    if case["kind"] == "read":
        _fill(case, state, g, start + t)
        return dict(state, start=start, counts=counts)
    views, keep, strides = _source(case, g)
    return dict(state, start=start, counts=counts, k=views[0], v=views[1], keep=keep, strides=strides)


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    b, t = case["b"], case["t"]
    if case["kind"] == "attention":
        state["out"] = torch.zeros_like(state["q"])
    else:
        half = case.get("dst") == "f16"
        shape = (b, case["hkv"], t, case["d"]) if case["kind"] == "read" and case["rows"] == "heads" else (b, t, case["hkv"], case["d"])
        state["outs"] = [torch.zeros(*shape, dtype=torch.float16 if half else torch.float32, device=DEV) for _ in "kv"]
    if own:
        _bind(case, state)
    torch.cuda.synchronize()
    return state


# ---- the framework's calls -------------------------------------------------------------

_stream = None


def _bind(case, state):
    """The case's entry points with their arguments."""
    from aljabr_amd import abi
    global _stream
    if _stream is None:
        abi.init(0)
        _stream = torch.cuda.Stream()
        abi.call("aljabr_rocm_set_stream", _stream.cuda_stream)
        abi.call("aljabr_rocm_set_sync_mode", 0)
    lib, table = abi.load(), state["table"]

    def at(x):
        return None if x is None else x.data_ptr()

    s, hkv, r = state["k_codes"].shape[:3]
    cache = abi.Kv4Cache(at(state["k_codes"]), at(state["k_scales"]), at(state["v_codes"]), at(state["v_scales"]), at(table),
                         case["b"], hkv, case["d"], r, s if table is not None else 0,
                         table.shape[1] if table is not None else 0)
    c, b, t, d = ctypes.byref(cache), case["b"], case["t"], case["d"]
    types = {"f32": abi.TYPE_F32, "f16": abi.TYPE_F16}
    calls = []
    if case["kind"] == "attention":
        calls.append(("aljabr_rocm_kv4_attention", at(state["out"]), at(state["q"]), c, at(state["lens"]), at(state["counts"]), t,
                      case["hq"], 0.0, 1, case["window"], case["softcap"], None, 0))
    else:
        start, counts, outs = at(state["start"]), at(state["counts"]), state["outs"]
        dense, heads = (t * hkv * d, hkv * d, d), (hkv * t * d, d, t * d)
        dst, strides = types["f32"], dense
        if case["kind"] == "write":
            calls.append(("aljabr_rocm_kv4_write", c, at(state["k"]), at(state["v"]), start, counts, t, *state["strides"],
                          types[case["src"]]))
        else:
            dst, strides = types[case["dst"]], heads if case["rows"] == "heads" else dense
        calls.append(("aljabr_rocm_kv4_read", at(outs[0]), at(outs[1]), c, start, counts, t, *strides, dst))
    state["calls"] = [(getattr(lib, n), n, a) for n, *a in calls]
    state["hold"] = cache


def _run_own(state):
    for fn, name, args in state["calls"]:
        rc = fn(*args)
        if rc:
            from aljabr_amd import abi
            abi.check(rc, name)
    return state["out"] if "out" in state else state["outs"]


# ---- one pass -----------------------------------------------------------------------------

def _visible(lens, counts, t, n, window):
    """Keys seen by row i of each sequence, [b, t, n], and the rows that exist, [b, t]."""
    cnt = counts.long() if counts is not None else torch.full_like(lens.long(), t)
    i = torch.arange(t, device=lens.device)[None]
    pos = lens.long()[:, None] - cnt[:, None] + i
    j = torch.arange(n, device=lens.device)
    see = j[None, None] <= torch.minimum(pos, lens.long()[:, None] - 1)[..., None]
    if window:
        see &= j[None, None] > (pos - window)[..., None]
    return see, i < cnt[:, None]


def _plain_attention(case, state):
    b, t, hq, hkv, d = (case[n] for n in ("b", "t", "hq", "hkv", "d"))
    n = case["ctx"]
    pos = torch.arange(n, device=DEV)[None].expand(b, n)
    pos = torch.minimum(pos, state["lens"].long()[:, None] - 1)       # rows past a sequence's end repeat its last, and are masked
    s, r = _row_index(state["table"], pos, case["page"])
    k = _gather(state, "k", s, r).permute(0, 2, 3, 1).contiguous()    # [b, hkv, d, n]
    q = state["q"].reshape(b, t, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    sc = torch.matmul(q * d ** -0.5, k).reshape(b, hkv, -1, t, n)
    del k
    if case["softcap"]:
        sc = case["softcap"] * torch.tanh(sc / case["softcap"])
    see, live = _visible(state["lens"], state["counts"], t, n, case["window"])
    sc = sc.masked_fill_(~see[:, None, None], -math.inf)
    top = sc.amax(-1, keepdim=True)
    sc = sc.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = sc.sum(-1, keepdim=True)
    v = _gather(state, "v", s, r).permute(0, 2, 1, 3).contiguous()
    out = torch.matmul(sc.reshape(b, hkv, -1, n), v).reshape(b, hkv, -1, t, d)
    out = torch.where(total > 0, out / total, 0.0).permute(0, 3, 1, 2, 4).reshape(b, t, hq, d)
    return torch.where(live[..., None, None], out, 0.0)


def _plain_rows(case, state):
    """Rows written (kind write) and read back."""
    b, t, page = case["b"], case["t"], case["page"]
    i = torch.arange(t, device=DEV)[None].expand(b, t)
    live = i < state["counts"].long()[:, None] if state["counts"] is not None else torch.ones_like(i, dtype=torch.bool)
    s, r = _row_index(state["table"], state["start"].long()[:, None] + i, page)
    outs = []
    for which in "kv":
        if case["kind"] == "write":
            scale, q = _scale_and_codes(state[which])
            state[which + "_codes"][s[live], :, r[live]] = _pack(q)[live]
            state[which + "_scales"][s[live], :, :, r[live]] = scale.half()[live]
        x = torch.where(live[..., None, None], _gather(state, which, s, r), 0.0)
        if case["kind"] == "read" and case["rows"] == "heads":
            x = x.transpose(1, 2)
        outs.append(x.half() if case.get("dst") == "f16" else x)
    return outs


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    return _plain_attention(case, state) if case["kind"] == "attention" else _plain_rows(case, state)


# ---- what a pass cannot do without -----------------------------------------------------------

def _pairs(case):
    """Visible (row, key) pairs, rows and keys of a case; ragged lengths are uniform in [1, ctx]."""
    b, t, ctx, window = (case[n] for n in ("b", "t", "ctx", "window"))
    full = [min(max(ctx - t + i + 1, 0), ctx) for i in range(t)]
    seen = sum(min(n, window) if window else n for n in full)
    keys = min(ctx, window + t - 1) if window else ctx
    if not case["ragged"]:
        return b * seen, b * t, b * keys
    # The first sequence is ctx long, and its row count uniform like the others'.
    part = (1 + (b - 1) / 2) * (1.0 if t == 1 else 0.5)
    if window and ctx > window:
        # The mean of min(len, window) over len in [1, ctx], against its largest value.
        mean = (window * (ctx - window / 2)) / ctx / window
        return (1 + (b - 1) * mean) * seen * (1.0 if t == 1 else 0.5), b * t * (1.0 if t == 1 else 0.5), (1 + (b - 1) * mean) * keys
    return part * seen, b * t * (1.0 if t == 1 else 0.5), (1 + (b - 1) / 2) * keys


def work(case):
    hkv, d = case["hkv"], case["d"]
    held = 0.5 + 2 / BLOCK                               # bytes an element in the cache
    if case["kind"] == "attention":
        pairs, rows, keys = _pairs(case)
        return {"bytes": 2 * held * keys * hkv * d + 8.0 * rows * case["hq"] * d, "flops": 4.0 * case["hq"] * d * pairs}
    b, t = case["b"], case["t"]
    rows = b * t if not case["ragged"] else t + (b - 1) * t / 2
    per = {"f32": 4, "f16": 2}
    if case["kind"] == "read":
        moved = held + per[case["dst"]]
    else:
        moved = per[case["src"]] + held + held + 4       # written, then read back as fp32
    return {"bytes": 2.0 * rows * hkv * d * moved, "flops": 2.0 * rows * hkv * d}


# ---- the same from the definition, in float64 ---------------------------------------------------

def _exact_values(x):
    """What a block of 32 is held as, of [..., d] rows, from the definition: a signed step of an eighth of the value
    of largest magnitude (the negative one of two alike) with 8 significant bits, and the nearest multiple of it."""
    x = x.double().unflatten(-1, (-1, BLOCK))
    low, high = x.min(-1).values, x.max(-1).values
    end = torch.maximum(high, -low)
    step = end / 8
    quantum = torch.exp2(torch.clamp(torch.floor(torch.log2(step.clamp(min=2.0 ** -60))) - 7, min=-24))
    step = torch.clamp(torch.round(step / quantum) * quantum, max=8160.0)
    step = torch.where(-low >= high, step, -step)
    n = torch.clamp(-torch.ceil(-x / step[..., None] - 0.5), -8, 7)
    return torch.where(step[..., None] == 0, torch.zeros_like(n), n * step[..., None]).flatten(-2)


def _exact_cached(state, which, b, n, page):
    """The first n rows of sequence b as float64 [heads, n, d]."""
    codes, scales = state[which + "_codes"], state[which + "_scales"]
    if page:
        blocks = state["table"][b, :-(-n // page)].long()
        codes = codes[blocks].transpose(0, 1).flatten(1, 2)[:, :n]
        scales = scales[blocks].permute(1, 2, 0, 3).flatten(2, 3)[:, :, :n]
    else:
        codes, scales = codes[b, :, :n], scales[b, :, :, :n]
    low, high = (codes % 16).double(), torch.div(codes, 16, rounding_mode="floor").double()
    c = torch.stack([low.unflatten(-1, (-1, 16)), high.unflatten(-1, (-1, 16))], -2).flatten(-2)     # [h, n, d/32, 32]
    return ((c - 8) * scales.double().transpose(1, 2)[..., None]).flatten(-2)


def _exact_attention(case, state):
    t, hq, hkv, d, window, cap = (case[n] for n in ("t", "hq", "hkv", "d", "window", "softcap"))
    out = torch.zeros_like(state["q"], dtype=torch.float64)
    for b, n in enumerate(state["lens"].tolist()):
        rows = t if state["counts"] is None else int(state["counts"][b])
        k, v = (_exact_cached(state, w, b, n, case["page"]) for w in "kv")
        last = n - rows + torch.arange(rows, device=DEV)
        keys = torch.arange(n, device=DEV)
        hidden = keys[None] > last[:, None]
        if window:
            hidden = hidden | (keys[None] <= last[:, None] - window)
        for h in range(hkv):
            heads = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
            q = state["q"][b, :rows, heads].double().reshape(-1, d)
            sc = (q @ k[h].t()).reshape(rows, -1, n) / math.sqrt(d)
            if cap:
                sc = cap * torch.tanh(sc / cap)
            p = torch.softmax(sc.masked_fill(hidden[:, None], -math.inf), -1)
            p = torch.nan_to_num(p) if bool(hidden.all(-1).any()) else p
            out[b, :rows, heads] = (p.reshape(-1, n) @ v[h]).reshape(rows, -1, d)
    return out


def exact(case, seed):
    state = _inputs(case, seed)
    if case["kind"] == "attention":
        return _exact_attention(case, state)
    b, t = case["b"], case["t"]
    counts = [t] * b if state["counts"] is None else state["counts"].tolist()
    outs = []
    for which in "kv":
        if case["kind"] == "write":
            x = _exact_values(state[which])
        else:
            x = torch.zeros(b, t, case["hkv"], case["d"], dtype=torch.float64, device=DEV)
            for s, start in enumerate(state["start"].tolist()):
                x[s] = _exact_cached(state, which, s, start + t, case["page"])[:, start:].transpose(0, 1)
        for s, n in enumerate(counts):
            x[s, n:] = 0
        outs.append(x.transpose(1, 2) if case["kind"] == "read" and case["rows"] == "heads" else x)
    return outs
