"""The operators of a decode step that verifies a tree of drafted tokens over a
cache of K and V rows, as this framework's speed in them is measured: rows
rotated and appended to the cache, attention of the tree's rows over it, and the
walk that accepts drafted tokens and moves their rows together.

K and V are planes [layers][S][heads][R][head_dim] of float16 or float32, with S
sequences of R rows (contiguous), or S blocks of R = block rows that a table
hands to sequences (paged).

A draft has t rows a sequence. Row i has a parent among the rows before it, or
-1; its depth is the number of its ancestors. The rows' places in the cache are
len - count + i, their positions len - count + depth. Without parents they are a
chain: the tokens of a plain decode step, or a chunk of a prompt.

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
VOCAB = 128256
BASE = 500000.0
TYPES = {"f16": torch.float16, "f32": torch.float32}


# ---- the cases --------------------------------------------------------------------

def listed():
    return [
        # One token of a Llama-3-8B layer at batch 1: launches are all there is.
        dict(name="append_token_b1", kind="append", b=1, t=1, hq=32, hkv=8, d=128, cap=2064, page=0, type="f16", src="f32",
             rows="dense", rot=128, inter=0, tree=0, far=0, divisors=0, ragged=0),
        # Trees of up to 26 drafts in 16 sequences, slices of the stacked Q/K/V product, a partly rotated head far into
        # a context with scaled frequencies, over a paged fp32 cache.
        dict(name="append_tree26_b16_paged", kind="append", b=16, t=26, hq=16, hkv=4, d=64, cap=2064, page=32, type="f32",
             src="f32", rows="qkv", rot=32, inter=1, tree=1, far=1000000, divisors=1, ragged=1),
        # Four prompts of up to 2048 tokens.
        dict(name="append_prompt_b4_2048", kind="append", b=4, t=2048, hq=32, hkv=8, d=128, cap=4096, page=16, type="f16",
             src="f32", rows="qkv", rot=128, inter=0, tree=0, far=0, divisors=0, ragged=1),
        # A tree of 8 drafts at batch 1 and short context: latency.
        dict(name="tree8_b1_512", kind="attention", b=1, t=8, hq=32, hkv=8, d=128, ctx=512, cap=2064, page=0, type="f16", tree=1,
             ragged=0, window=0, softcap=0.0),
        # A serving batch: 32 sequences of every length up to 4096, chains of up to five drafts, pages of 16.
        dict(name="chain5_b32_ragged_paged", kind="attention", b=32, t=5, hq=32, hkv=8, d=128, ctx=4096, cap=4112, page=16,
             type="f16", tree=0, ragged=1, window=0, softcap=0.0),
        # Trees of 64 drafts in 8 sequences of 8192 keys.
        dict(name="tree64_b8_8192_paged", kind="attention", b=8, t=64, hq=32, hkv=8, d=128, ctx=8192, cap=8192, page=64,
             type="f16", tree=1, ragged=0, window=0, softcap=0.0),
        # A tree of 26 drafts over one very long context.
        dict(name="tree26_b1_131072", kind="attention", b=1, t=26, hq=32, hkv=8, d=128, ctx=131072, cap=131072, page=0,
             type="f16", tree=1, ragged=0, window=0, softcap=0.0),
        # Heads of 256 with a sliding window and a soft cap, trees of up to 12.
        dict(name="tree12_b4_window_d256", kind="attention", b=4, t=12, hq=16, hkv=8, d=256, ctx=4096, cap=4112, page=64,
             type="f16", tree=1, ragged=1, window=1024, softcap=50.0),
        # Trees of 16 over a paged fp32 cache.
        dict(name="tree16_b4_2048_f32", kind="attention", b=4, t=16, hq=32, hkv=8, d=128, ctx=2048, cap=2064, page=16, type="f32",
             tree=1, ragged=0, window=0, softcap=0.0),
        # Two 512-token chunks of prompts against the earlier chunks in the paged cache.
        dict(name="chunk512_b2_4096", kind="attention", b=2, t=512, hq=32, hkv=8, d=128, ctx=4096, cap=4096, page=16, type="f16",
             tree=0, ragged=0, window=0, softcap=0.0),
        # What a tree of 64 at batch 1 leaves in the cache of a 32-layer session.
        dict(name="accept_tree64_b1", kind="accept", b=1, t=64, hkv=8, d=128, ctx=200, cap=272, page=0, type="f16", layers=32,
             keep=7, ragged=0),
        # The same for 32 sequences of a paged cache.
        dict(name="accept_tree26_b32_paged", kind="accept", b=32, t=26, hkv=8, d=128, ctx=96, cap=128, page=16, type="f16",
             layers=16, keep=6, ragged=1),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    """Another case of the listed ranges: any batch up to 64, drafts of one row
    to trees of 256 and chunks of 1024, contexts from one key to 131072, heads
    of 64, 128 and 256 in any grouping, fp16 and fp32 caches, contiguous ones of
    any length and pages of 16 to 128 rows."""
    kind = rng.choice(["append", "append", "attention", "attention", "attention", "attention", "accept"])
    d = rng.choice([64, 128, 128, 256])
    page = rng.choice([0, 0, 16, 32, 64, 128])
    typ = rng.choice(["f16", "f16", "f32"])
    hkv, g = rng.choice([(8, 4), (8, 4), (8, 8), (4, 8), (8, 1), (16, 2), (4, 7), (2, 3), (1, 16), (2, 12)])
    if kind == "append":
        b = rng.choice([1, _log(rng, 2, 64)])
        tree = rng.choice([0, 1])
        t = rng.randint(2, 64) if tree else 1 if rng.random() < 0.3 else _log(rng, 2, 8192 // b)
        t = max(1, min(t, (1 << 23) // (b * hkv * g * d) * 4))
        rot = d if rng.random() < 0.6 else 8 * rng.randint(1, d // 8)
        return dict(kind=kind, b=b, t=t, hq=hkv * g, hkv=hkv, d=d, cap=t + rng.choice([0, 15, 100]), page=page, type=typ,
                    src=rng.choice(["f32", "f32", "f16"]), rows=rng.choice(["dense", "qkv", "heads"]), rot=rot,
                    inter=rng.choice([0, 0, 1]), tree=tree, far=rng.choice([0, 0, 100000, 1000000]),
                    divisors=rng.choice([0, 1]), ragged=rng.choice([0, 1]))
    if kind == "accept":
        t = _log(rng, 2, 256)
        b, layers = _log(rng, 1, 32), rng.choice([1, 7, 16, 32])
        b = max(1, min(b, (1 << 27) // (layers * hkv * d * (t + 40))))
        return dict(kind=kind, b=b, t=t, hkv=hkv, d=d, ctx=t + rng.randint(0, 20), cap=t + rng.randint(20, 40), page=page, type=typ,
                    layers=layers, keep=rng.randint(1, min(t, 16)), ragged=rng.choice([0, 1]))
    window, cap50 = rng.choice([(0, 0.0), (0, 0.0), (0, 0.0), (_log(rng, 2, 2048), 0.0), (1024, 50.0)])
    form = rng.choice(["decode", "chain", "tree", "tree", "tree", "chunk"])
    t = {"decode": 1, "chain": rng.randint(2, 8), "tree": _log(rng, 2, 256 if rng.random() < 0.2 else 64),
         "chunk": _log(rng, 9, 1024)}[form]
    keys = (1 << 27) // (hkv * d * (2 if typ == "f32" else 1))
    pairs = (1 << 34) // (hkv * g * d * t)             # what bounds the products' operations
    ctx = min(keys, pairs, t + _log(rng, 1, 4096 if form == "chunk" else 131072) - 1)
    t = min(t, ctx)
    b = max(1, min(_log(rng, 1, 64), keys // ctx, pairs // ctx))
    return dict(kind=kind, b=b, t=t, hq=hkv * g, hkv=hkv, d=d, ctx=ctx, cap=ctx + rng.choice([0, 15, 100]), page=page, type=typ,
                tree=int(form == "tree"), ragged=rng.choice([0, 1]), window=window, softcap=cap50)


# ---- what a program has in hand before the call --------------------------------------

class _Draw:
    """Seeded tensors on the device."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV).manual_seed(int(seed))

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.g, device=DEV)

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.g, device=DEV)

    def ints(self, lo, hi, *shape):
        return torch.randint(lo, hi + 1, shape, generator=self.g, device=DEV, dtype=torch.int32)


def _planes(case, g, lens):
    """The case's K and V planes, filled, and its table: blocks in shuffled order, -1 past a sequence's last."""
    b, hkv, d, cap, page = (case[n] for n in ("b", "hkv", "d", "cap", "page"))
    s, r, table = b, cap, None
    if page:
        per = -(-cap // page)
        s, r = b * per + 3, page
        table = torch.randperm(s, generator=g.g, device=DEV)[:b * per].int().reshape(b, per)
        used = (lens.long() + page - 1) // page
        table = torch.where(torch.arange(per, device=DEV)[None] < used[:, None], table, -1).int().contiguous()
    spread = torch.exp(0.5 * g.normal(hkv, 1, d))       # keys with the uneven channels that they have
    shape = (case.get("layers", 1), s, hkv, r, d)
    state = {"table": table}
    for which in "kv":
        x = torch.empty(shape, dtype=TYPES[case["type"]], device=DEV)
        for layer in x:
            for i in range(0, s, 1024):
                y = g.normal(*layer[i:i + 1024].shape)
                layer[i:i + 1024] = y * spread if which == "k" else y
        state[which] = x
    return state


def _parents(g, b, t):
    """Trees with more children near the root: row i's parent is before it, row 0 has none."""
    i = torch.arange(t, device=DEV)
    p = (g.uniform(b, t) ** 2 * i).int().clamp_(max=max(t - 2, 0))
    return torch.where(i == 0, -1, torch.minimum(p, (i - 1).clamp(min=0).int())).int().contiguous()


def _rows_of(case, g):
    """Q, K and V rows [b, t, heads, d] as the program holds them, and Q's and K's strides (sequence, token, head)."""
    b, t, hq, hkv, d = (case[n] for n in ("b", "t", "hq", "hkv", "d"))
    dtype = TYPES[case["src"]]
    if case["rows"] == "qkv":
        x = g.normal(b, t, hq + 2 * hkv, d).to(dtype)
        row = (hq + 2 * hkv) * d
        return (x[:, :, :hq], x[:, :, hq:hq + hkv], x[:, :, hq + hkv:]), ((t * row, row, d),) * 2
    if case["rows"] == "heads":
        x = [g.normal(b, n, t, d).to(dtype).transpose(1, 2) for n in (hq, hkv, hkv)]
        return tuple(x), ((hq * t * d, d, t * d), (hkv * t * d, d, t * d))
    x = [g.normal(b, t, n, d).to(dtype) for n in (hq, hkv, hkv)]
    return tuple(x), ((t * hq * d, hq * d, d), (t * hkv * d, hkv * d, d))


def _inputs(case, seed):
    """Everything of a case that the seed decides."""
    g, b, t = _Draw(seed), case["b"], case["t"]
    if case["kind"] == "append":
        start = g.ints(0, case["cap"] - t, b)
        counts = g.ints(0, t, b) if case["ragged"] else None
        if counts is not None:
            counts[0] = t
        state = dict(_planes(case, g, start + t), start=start, counts=counts)
        state["qkv"], state["strides"] = _rows_of(case, g)
        state["angles"] = None
        if case["tree"] or case["far"]:
            depth = _ancestors(_parents(g, b, t)).sum(-1) - 1 if case["tree"] else torch.arange(t, device=DEV)
            state["angles"] = (start[:, None] + depth + case["far"]).int().contiguous()
        state["divisors"] = 1 + 7 * g.uniform(case["rot"] // 2) if case["divisors"] else None
        return state
    lens = g.ints(1, case["ctx"], b) if case["ragged"] else torch.full((b,), case["ctx"], dtype=torch.int32, device=DEV)
    lens[0] = case["ctx"]
    # A draft is padded to t rows: the last `counts` places belong to its rows.
    counts = torch.minimum(g.ints(1, t, b), lens) if case["ragged"] and t > 1 else None
    if counts is None:
        lens = lens.clamp(min=t)
    state = dict(_planes(case, g, lens), lens=lens, counts=counts)
    if case["kind"] == "attention":
        state["parents"] = _parents(g, b, t) if case["tree"] else None
        state["q"] = g.normal(b, t, case["hq"], case["d"])
        return state
    # A path of up to `keep` rows on which the model agrees with the draft, among rows of which it does not.
    keep = g.ints(1, case["keep"], b) if case["ragged"] else torch.full((b,), case["keep"], dtype=torch.int32, device=DEV)
    n = case["keep"]
    spine = torch.argsort(g.uniform(b, t - 1), -1)[:, :n - 1].sort(-1).values + 1
    spine = torch.cat([torch.zeros(b, 1, dtype=torch.long, device=DEV), spine], -1)
    parents = _parents(g, b, t)
    parents.scatter_(1, spine[:, 1:], spine[:, :-1].int())
    tokens, choices = g.ints(0, VOCAB - 1, b, t), g.ints(0, VOCAB - 1, b, t)
    agree = torch.where(torch.arange(1, n, device=DEV)[None] < keep[:, None], torch.gather(tokens, 1, spine[:, 1:]), -1)
    choices.scatter_(1, spine[:, :-1], agree.int())
    return dict(state, parents=parents, tokens=tokens, choices=choices)


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    b, t = case["b"], case["t"]
    if case["kind"] == "attention":
        state["out"] = torch.zeros_like(state["q"])
    elif case["kind"] == "append":
        state["q_out"] = torch.zeros(b, t, case["hq"], case["d"], device=DEV)
    else:
        state["path"] = torch.zeros(b, t, dtype=torch.int32, device=DEV)
        for name in ("new_lens", "accepted", "next"):
            state[name] = torch.zeros(b, dtype=torch.int32, device=DEV)
    if own:
        _bind(case, state)
    torch.cuda.synchronize()
    return state


# ---- the framework's calls -------------------------------------------------------------

_stream = None


def _bind(case, state):
    """The case's entry point with its arguments."""
    from aljabr_amd import abi
    global _stream
    if _stream is None:
        abi.init(0)
        _stream = torch.cuda.Stream()
        abi.call("aljabr_rocm_set_stream", _stream.cuda_stream)
        abi.call("aljabr_rocm_set_sync_mode", 0)
    table = state["table"]

    def at(x):
        return None if x is None else x.data_ptr()

    types = {"f32": abi.TYPE_F32, "f16": abi.TYPE_F16}
    layers, s, hkv, r, d = state["k"].shape
    cache = abi.KvCache(at(state["k"]), at(state["v"]), at(table), types[case["type"]], layers, case["b"], hkv, d, r,
                        s if table is not None else 0, table.shape[1] if table is not None else 0)
    c, t = ctypes.byref(cache), case["t"]
    if case["kind"] == "attention":
        name, args = "aljabr_rocm_kv_tree_attention", (
            at(state["out"]), at(state["q"]), c, 0, at(state["lens"]), at(state["counts"]), at(state["parents"]), t, case["hq"],
            0.0, case["window"], case["softcap"], None, 0)
        state["answer"] = state["out"]
    elif case["kind"] == "append":
        rotation = abi.Rotation(BASE, case["rot"], case["inter"], at(state["divisors"]))
        q, k, v = state["qkv"]
        name, args = "aljabr_rocm_kv_append", (
            c, 0, at(state["q_out"]), at(q), at(k), at(v), at(state["start"]), at(state["counts"]), at(state["angles"]), t,
            case["hq"], *state["strides"][0], *state["strides"][1], types[case["src"]], ctypes.byref(rotation))
        state["answer"] = [state["q_out"], state["k"], state["v"]]
        state["hold_rotation"] = rotation
    else:
        name, args = "aljabr_rocm_kv_tree_accept", (
            c, at(state["new_lens"]), at(state["path"]), at(state["accepted"]), at(state["next"]), at(state["lens"]),
            at(state["counts"]), at(state["parents"]), at(state["tokens"]), at(state["choices"]), t)
        state["answer"] = [state[n] for n in ("new_lens", "path", "accepted", "next", "k", "v")]
    state["call"] = (getattr(abi.load(), name), name, args)
    state["hold"] = cache


def _run_own(state):
    fn, name, args = state["call"]
    rc = fn(*args)
    if rc:
        from aljabr_amd import abi
        abi.check(rc, name)
    return state["answer"]


# ---- one pass in plain torch --------------------------------------------------------------

def _row_index(table, pos, page):
    """The (sequence or block, row) of positions pos [b, t]."""
    if table is None:
        return torch.arange(pos.shape[0], device=pos.device)[:, None].expand_as(pos), pos
    return torch.gather(table.long(), 1, pos // page), pos % page


def _ancestors(parents):
    """[b, t, t]: row i is row t or one of its ancestors."""
    t = parents.shape[1]
    i = torch.arange(t, device=DEV)
    near = ((parents.long()[..., None] == i) | (i[:, None] == i)).float()
    for _ in range(max(t - 1, 1).bit_length()):
        near = torch.matmul(near, near).clamp_(max=1)
    return near > 0.5


def _live(case, state):
    """The rows' count of each sequence and whether row i exists, [b], [b, t]."""
    b, t = case["b"], case["t"]
    counts = state["counts"].long() if state["counts"] is not None else torch.full((b,), t, device=DEV)
    return counts, torch.arange(t, device=DEV)[None] < counts[:, None]


def _rotate(case, state, x):
    """[b, t, heads, d] float32 rotated; the angles are computed in 64 bits."""
    rot, t = case["rot"], case["t"]
    a = state["angles"] if state["angles"] is not None else state["start"][:, None] + torch.arange(t, device=DEV)
    freq = BASE ** (-2.0 * torch.arange(rot // 2, device=DEV, dtype=torch.float64) / rot)
    if state["divisors"] is not None:
        freq = freq / state["divisors"].double()
    theta = a.double()[..., None, None] * freq
    c, s = torch.cos(theta).float(), torch.sin(theta).float()
    if case["inter"]:
        x0, x1 = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack([x0 * c - x1 * s, x0 * s + x1 * c], -1).flatten(-2)
    else:
        x0, x1 = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat([x0 * c - x1 * s, x0 * s + x1 * c], -1)
    return torch.cat([y, x[..., rot:]], -1)


def _plain_append(case, state):
    _, live = _live(case, state)
    q, k, v = (x.float() for x in state["qkv"])
    q, k = _rotate(case, state, q), _rotate(case, state, k)
    state["q_out"][live] = q[live]
    pos = state["start"].long()[:, None] + torch.arange(case["t"], device=DEV)
    s, r = _row_index(state["table"], pos, case["page"])
    for which, x in (("k", k), ("v", v)):
        state[which][0][s[live], :, r[live]] = x[live].to(state[which].dtype)
    return [state["q_out"], state["k"], state["v"]]


def _plain_attention(case, state):
    b, t, hq, hkv, d, window = (case[n] for n in ("b", "t", "hq", "hkv", "d", "window"))
    n = case["ctx"]
    lens = state["lens"].long()
    counts, live = _live(case, state)
    base = lens - counts
    pos = torch.arange(n, device=DEV)[None].expand(b, n)
    s, r = _row_index(state["table"], torch.minimum(pos, lens[:, None] - 1), case["page"])   # past the end: masked
    k = state["k"][0][s, :, r].float().permute(0, 2, 3, 1).contiguous()                      # [b, hkv, d, n]
    q = state["q"].reshape(b, t, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    sc = torch.matmul(q * d ** -0.5, k).reshape(b, hkv, -1, t, n)
    del k
    if case["softcap"]:
        sc = case["softcap"] * torch.tanh(sc / case["softcap"])
    # Key j is a cached one, or row j - base of the draft, which sees it or not.
    i = torch.arange(t, device=DEV)
    mine = _ancestors(state["parents"]) if case["tree"] else (i[:, None] >= i).expand(b, t, t)
    depth = mine.sum(-1) - 1
    of_draft = pos - base[:, None]
    row = of_draft.clamp(0, t - 1)[:, None].expand(b, t, n)
    see = torch.where(of_draft[:, None] < 0, True, torch.gather(mine, 2, row) & (of_draft < counts[:, None])[:, None])
    if window:
        key = torch.where(of_draft < 0, of_draft, torch.gather(depth, 1, row[:, 0]))
        see &= depth[..., None] - key[:, None] < window
    sc = sc.masked_fill_(~see[:, None, None], -math.inf)
    top = sc.amax(-1, keepdim=True)
    sc = sc.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = sc.sum(-1, keepdim=True)
    v = state["v"][0][s, :, r].float().permute(0, 2, 1, 3).contiguous()
    out = torch.matmul(sc.reshape(b, hkv, -1, n), v).reshape(b, hkv, -1, t, d)
    out = torch.where(total > 0, out / total, 0.0).permute(0, 3, 1, 2, 4).reshape(b, t, hq, d)
    return torch.where(live[..., None, None], out, 0.0)


def _plain_accept(case, state):
    b, t = case["b"], case["t"]
    counts, live = _live(case, state)
    base = state["lens"].long() - counts
    i = torch.arange(t, device=DEV)
    up = state["parents"].long().clamp(min=0)
    agreed = live & (state["parents"] >= 0) & (state["tokens"] == torch.gather(state["choices"], 1, up))
    # Of a row's children that agree the first counts.
    twin = agreed[:, :, None] & agreed[:, None] & (up[:, :, None] == up[:, None]) & (i[None, :, None] > i)
    agreed = agreed & ~twin.any(-1)
    agreed[:, 0] = live[:, 0]
    mine = _ancestors(state["parents"])
    kept = mine[:, :, 0] & (agreed[:, None] | ~mine).all(-1)
    order = torch.where(kept, i, t).sort(-1).values
    state["path"].copy_(torch.where(order < t, order, -1))
    m = kept.sum(-1)
    state["accepted"].copy_(m)
    state["new_lens"].copy_(base + m)
    last = torch.gather(state["path"].long(), 1, (m - 1).clamp(min=0)[:, None]).clamp(min=0)
    state["next"].copy_(torch.where(m > 0, torch.gather(state["choices"], 1, last)[:, 0], -1))
    moved = order < t
    sb, sr = _row_index(state["table"], torch.where(moved, base[:, None] + order, 0), case["page"])
    tb, tr = _row_index(state["table"], torch.where(moved, base[:, None] + i, 0), case["page"])
    for which in "kv":
        rows = state[which][:, sb[moved], :, sr[moved]]
        state[which][:, tb[moved], :, tr[moved]] = rows
    return [state[n] for n in ("new_lens", "path", "accepted", "next", "k", "v")]


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    return {"append": _plain_append, "attention": _plain_attention, "accept": _plain_accept}[case["kind"]](case, state)


# ---- what a pass cannot do without -----------------------------------------------------------

def work(case):
    """Ragged lengths are uniform in [1, ctx], counts in [1, t] (appended ones in [0, t])."""
    b, t, hkv, d = (case[n] for n in ("b", "t", "hkv", "d"))
    size = {"f16": 2, "f32": 4}[case["type"]]
    mean = (b + 1) / 2 if case["ragged"] else b             # sequences of full length that they come to
    if case["kind"] == "append":
        rows, src = t * mean, {"f16": 2, "f32": 4}[case["src"]]
        return {"bytes": rows * d * (case["hq"] * (src + 4.0) + 2 * hkv * (src + size)),
                "flops": 3.0 * rows * case["rot"] * (case["hq"] + hkv)}
    if case["kind"] == "accept":
        kept = (case["keep"] + 1) / 2 if case["ragged"] else case["keep"]
        return {"bytes": 4.0 * case["layers"] * b * (kept - 1) * hkv * d * size + 16.0 * b * t, "flops": 4.0 * b * t}
    ctx, window = case["ctx"], case["window"]
    rows = t * (b / 2 if case["ragged"] and t > 1 else b)
    keys = ctx * mean
    if window and ctx > window:
        # The mean of min(len, window) over len in [1, ctx].
        keys = window * (1 + (b - 1) * (1 - window / (2 * ctx))) if case["ragged"] else window * b
    return {"bytes": 2.0 * size * keys * hkv * d + 8.0 * rows * case["hq"] * d,
            "flops": 4.0 * case["hq"] * d * (rows / b) * keys}


# ---- the same from the definition, in float64 ---------------------------------------------------

def _place(state, case, b, j):
    """Where key j of sequence b is: (plane, row)."""
    if state["table"] is None:
        return b, j
    return int(state["table"][b, j // case["page"]]), j % case["page"]


def _exact_cached(state, case, which, b, n):
    """The first n rows of sequence b as float64 [heads, n, d]."""
    x = state[which][0]
    if state["table"] is None:
        return x[b, :, :n].double()
    blocks = state["table"][b, :-(-n // case["page"])].long()
    return x[blocks].transpose(0, 1).flatten(1, 2)[:, :n].double()


def _exact_append(case, state):
    t, rot = case["t"], case["rot"]
    q, k, v = (x.double() for x in state["qkv"])
    out = {"q": torch.zeros_like(q), "k": state["k"].double(), "v": state["v"].double()}
    power = torch.arange(0, rot, 2, device=DEV).double() / rot
    for b, start in enumerate(state["start"].tolist()):
        n = t if state["counts"] is None else int(state["counts"][b])
        if not n:
            continue
        at = start + torch.arange(n, device=DEV) if state["angles"] is None else state["angles"][b, :n]
        angle = at.double()[:, None] * torch.exp(-power * math.log(BASE))[None]
        if state["divisors"] is not None:
            angle = angle / state["divisors"].double()
        turn = torch.polar(torch.ones_like(angle), angle)[:, None]
        rows = {"v": v[b, :n]}
        for name, x in (("q", q[b, :n]), ("k", k[b, :n])):
            # Pairs as complex numbers, turned.
            pairs = x[..., :rot].unflatten(-1, (-1, 2) if case["inter"] else (2, -1))
            z = torch.complex(pairs[..., 0], pairs[..., 1]) if case["inter"] else torch.complex(pairs[..., 0, :], pairs[..., 1, :])
            z = z * turn
            y = torch.view_as_real(z)
            rows[name] = torch.cat([y.flatten(-2) if case["inter"] else y.transpose(-1, -2).flatten(-2), x[..., rot:]], -1)
        out["q"][b, :n] = rows["q"]
        pos = torch.arange(start, start + n, device=DEV)
        plane = torch.full_like(pos, b) if state["table"] is None else state["table"][b].long()[pos // case["page"]]
        place = pos if state["table"] is None else pos % case["page"]
        for name in "kv":
            out[name][0, plane, :, place] = rows[name]
    return [out["q"], out["k"], out["v"]]


def _exact_attention(case, state):
    t, hq, hkv, d, window, cap = (case[n] for n in ("t", "hq", "hkv", "d", "window", "softcap"))
    out = torch.zeros_like(state["q"], dtype=torch.float64)
    for b, n in enumerate(state["lens"].tolist()):
        rows = t if state["counts"] is None else int(state["counts"][b])
        base = n - rows
        hidden = torch.ones(rows, n, dtype=torch.bool)
        up = list(range(-1, rows - 1)) if not case["tree"] else state["parents"][b].tolist()
        depth = []
        for r in range(rows):
            depth.append(0 if up[r] < 0 else depth[up[r]] + 1)
            hidden[r, :base] = False
            i, steps = r, 0
            while i >= 0 and (not window or steps < window):
                hidden[r, base + i] = False
                i, steps = up[i], steps + 1
            if window:
                hidden[r, :max(0, min(base, base + depth[r] - window + 1))] = True
        hidden = hidden.to(DEV)
        k, v = (_exact_cached(state, case, w, b, n) for w in "kv")
        for h in range(hkv):
            heads = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
            q = state["q"][b, :rows, heads].double().reshape(-1, d)
            sc = (q @ k[h].t()).reshape(rows, -1, n) / math.sqrt(d)
            if cap:
                sc = cap * torch.tanh(sc / cap)
            p = torch.softmax(sc.masked_fill(hidden[:, None], -math.inf), -1)
            out[b, :rows, heads] = (p.reshape(-1, n) @ v[h]).reshape(rows, -1, d)
    return out


def _exact_accept(case, state):
    new_lens, accepted, after = [], [], []
    path = torch.full((case["b"], case["t"]), -1, dtype=torch.int32)
    k, v = state["k"].double(), state["v"].double()
    for b, n in enumerate(state["lens"].tolist()):
        rows = case["t"] if state["counts"] is None else int(state["counts"][b])
        up, tokens, choices = (state[w][b].tolist() for w in ("parents", "tokens", "choices"))
        walk = [0] if rows else []
        while walk:
            on = [i for i in range(rows) if up[i] == walk[-1] and tokens[i] == choices[walk[-1]]]
            if not on:
                break
            walk.append(on[0])
        path[b, :len(walk)] = torch.tensor(walk, dtype=torch.int32)
        accepted.append(len(walk))
        new_lens.append(n - rows + len(walk))
        after.append(choices[walk[-1]] if walk else -1)
        for i, r in enumerate(walk):                     # i <= r, and rows move forward in order
            (ps, rs), (pd, rd) = (_place(state, case, b, n - rows + j) for j in (r, i))
            for x in (k, v):
                x[:, pd, :, rd] = x[:, ps, :, rs].clone()
    whole = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in (new_lens, accepted, after)]
    return [whole[0], path.to(DEV), whole[1], whole[2], k, v]


def exact(case, seed):
    state = _inputs(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "accept": _exact_accept}[case["kind"]](case, state)
