// kv_tree.hpp - what the kernels of attention over fp16 and fp32 caches share:
// the rows' key ranges, their lines in a tree, where a tile's keys are.
// Included by the kv_tree .hip files only.
#pragma once

#include <algorithm>

#include "device.hpp"
#include "internal.hpp"
#include "kv_cache.hpp"
#include "kv_chunks.hpp"

namespace aljabr {
namespace kvt {

using namespace kv;

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256, kWaves = 4;
constexpr int kRowsBlock = 128;              // rows a workgroup of the rows kernel stacks
constexpr int kRowsLeast = 4;                // tiles it takes at the least
constexpr float kLog2e = 1.4426950408889634f;
// The reference that weights are relative to is raised only when a score (times log2(e)) exceeds it by more than kRaise:
// weights are at most 2^kRaise, and are kept times kWeightScale, as two fp16 parts that keep what is not below 2^-36 of the
// row's largest. (Raised at 2, with weights times 2^13: 2^-38, and a fifth more of the vector work in the rows kernel.)
constexpr float kRaise = 4.0f;
template <bool F16>
constexpr float kWeightScale = F16 ? 2048.0f : 1.0f;

struct Params {
    static constexpr bool kEvenChunks = true;
    KvView v;
    float *out;
    const float *q;
    const int *lens, *counts, *parents;
    int T, Hq, G, row_groups;
    FastDiv by_g, by_rows, by_chunks, by_heads, by_groups;             // G, rows of a block, quota (or sequences), H, row_groups
    int span_shift;                          // see work_at
    float scale, unscale;                    // their product is the call's scale times log2(e)
    int least_exp;                           // of a scaled query row's largest, see query_exponent
    float soft_cap;
    int window;
    int tile_shift;                          // log2 of the keys of a tile
    int quota;                               // chunks that the keys of all sequences are cut into (about), 0: one each
    float *part_o, *part_ml;                 // per slot, KV head, row group and stacked row: D sums, and (m, l)
    int2 *chunks;                            // per sequence, KV head and row group: its first slot and its chunks
};

// The rows lie where the length says, also past the cache's end, where it has no keys: base + cnt may exceed n.
__device__ __forceinline__ Seq sequence(const Params &p, int b) {
    Seq s;
    const int len = max(p.lens[b], 0);
    s.n = min(len, kv_capacity(p.v));
    s.cnt = p.counts ? min(max(p.counts[b], 0), p.T) : p.T;
    s.base = len - s.cnt;
    return s;
}

// Workgroups of the row groups that read the same keys are 2^span_shift numbers apart: 8, which is the same XCD (and its
// L2) at the same time, where there is enough to share out among the XCDs so. 256 rows over 8 sequences of 8192 keys 161 ->
// 156 us, over 32 of 4096 300 -> 287, against row groups H * quota numbers apart.
struct Work {
    int kvh, group, w;
};
__device__ __forceinline__ Work work_at(const Params &p, int id) {
    const int rest = id >> p.span_shift, q = p.by_groups(rest), u = (q << p.span_shift) + (id & ((1 << p.span_shift) - 1));
    Work x;
    x.group = rest - q * p.row_groups;
    x.w = p.by_heads(u);
    x.kvh = u - x.w * p.v.H;
    return x;
}
inline unsigned workgroups(const Params &p) {
    const int n = p.v.H * (p.quota ? p.quota + (p.v.B > 1 ? p.v.B : 0) : p.v.B), span = 1 << p.span_shift;
    return static_cast<unsigned>((n + span - 1) / span * span * p.row_groups);
}

// Numbers KV heads and row groups for partials.
__device__ __forceinline__ int item_of(const Params &p, int kvh, int group) { return group * p.v.H + kvh; }

// The first position less than `window` before the one in front of `next`; 0 without a window. No number leaves 32 bits: a
// position may be anything up to 2^31 - 2, and, with more rows than keys, below 0.
__device__ __forceinline__ int window_start(const Params &p, int next) {
    return p.window > 0 && next > p.window ? next - p.window : 0;
}

// The e with which an fp16 cache's query row, times p.scale, is scaled by 2^(15 - e): its largest magnitude `top` is in
// [2^(e-1), 2^e). Not less than p.least_exp, so that what scales the scores back, p.unscale 2^(e - 15), stays a normal number:
// zero times a masked key's -inf would be NaN. Scores so small weigh all keys alike.
__device__ __forceinline__ int query_exponent(const Params &p, float top) {
    int e = 0;
    if (top > 0.0f && top <= 3.4028235e38f) (void)frexpf(top, &e);
    return max(e, p.least_exp);
}

// The tiles that rows [r0, r0 + rows) see together. A row of a tree may stand anywhere between its root and its place,
// so the window is taken from the root and the last key from the place.
__device__ __forceinline__ bool row_tiles(const Params &p, const Seq &s, int r0, int rows, int &a, int &z) {
    a = z = 0;
    if (r0 >= s.cnt * p.G) return false;
    const int hi = min(s.base + min(p.by_g(r0 + rows - 1), s.cnt - 1) + 1, s.n);
    const int lo = window_start(p, s.base + (p.parents ? 0 : p.by_g(r0)) + 1);
    if (hi > lo) {                                           // else no tile, which past the end would not be there
        a = lo >> p.tile_shift;
        z = (hi + (1 << p.tile_shift) - 1) >> p.tile_shift;
    }
    return true;
}

// What a row sees: keys [lo, hi), and of a tree's rows those in its line.
struct Range {
    int lo, hi;
};
__device__ __forceinline__ Range range_of(const Params &p, const Seq &s, int t, const Tree &tree, bool filled) {
    Range x;
    x.hi = min(max(p.parents ? s.base : s.base + t + 1, 0), s.n);
    x.lo = window_start(p, s.base + (p.parents ? (filled ? tree.depth[t] : 0) : t) + 1);
    return x;
}

// Bits of keys k0 .. k0 + 31 that row t sees.
__device__ __forceinline__ uint32_t seen(const Params &p, const Seq &s, const Range &x, int t, int k0, const Tree &tree) {
    const int a = max(x.lo - k0, 0), z = min(x.hi - k0, 32);
    uint32_t bits = z <= a ? 0 : (z == 32 ? 0xffffffffu : (1u << z) - 1) & ~((1u << a) - 1);
    if (p.parents) {
        const int at = k0 - s.base;                          // of the tree's rows
        if (at >= 0 && at < s.cnt) {
            const int w = at >> 5;
            bits |= funnel_shift_right(w + 1 < kTreeWords ? tree.mask[(w + 1) * kTreeMost + t] : 0, tree.mask[w * kTreeMost + t], at & 31);
        } else if (at < 0 && at > -32) {
            bits |= tree.mask[t] << -at;
        }
        if (s.n - k0 < 32) bits &= (1u << (s.n - k0)) - 1;   // rows past the end
    }
    return bits;
}

// Where the groups of 16 keys of a wave's tiles first, first + step, .. are: lane i holds the byte offset of group i % U
// of the wave's tile i / U, 64 groups at once, so that a tile's address costs two lane reads and waits for no load.
template <int U>
struct Places {
    int first, step, held;                   // the wave's tiles [held, held + 64 / U) are held
    int lo, hi;                              // this lane's offset
    uint64_t there;                          // lanes whose group's block exists

    // What the table says of this lane's group, from the wave's i-th tile on: the block, or the sequence without a table.
    struct Entry {
        int s, row;
    };
    __device__ __forceinline__ Entry fetch(const Params &p, int lane, int b, int n_keys, int i) const {
        const long long tile = (first + static_cast<long long>(i + lane / U) * step) * (16 * U), last = n_keys - 1;
        long long key = tile + 16 * (lane % U);              // past the end: the tile's first group again, masked; or any
        if (key > last) key = tile;
        if (key > last) key = max(last, 0LL) & ~15;
        Entry x{b, static_cast<int>(key)};
        if (p.v.table) {
            const int blk = p.by_rows(x.row);
            x.s = p.v.table[static_cast<long long>(b) * p.v.max_blocks + blk];
            x.row -= blk * p.v.R;
        }
        return x;
    }
    __device__ __forceinline__ void hold(const Params &p, Entry x, int row_bytes, int kvh, int i) {
        held = i;
        const bool ok = !p.v.table || (x.s >= 0 && x.s < p.v.num_blocks);
        const long long at = ((static_cast<long long>(ok ? x.s : 0) * p.v.H + kvh) * p.v.R + x.row) * row_bytes;
        lo = static_cast<int>(at);
        hi = static_cast<int>(at >> 32);
        there = __ballot(ok);
    }
    __device__ __forceinline__ void load(const Params &p, int lane, int row_bytes, int b, int kvh, int n_keys, int i) {
        hold(p, fetch(p, lane, b, n_keys, i), row_bytes, kvh, i);
    }
    // Group u of the wave's i-th tile.
    __device__ __forceinline__ long long offset(int i, int u) const {
        const int l = (i - held) * U + u;
        return static_cast<long long>(static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(hi, l))) << 32 |
                                      static_cast<uint32_t>(__builtin_amdgcn_readlane(lo, l)));
    }
    // Bit u: group u's block exists.
    __device__ __forceinline__ uint32_t ok(int i) const {
        return static_cast<uint32_t>(there >> ((i - held) * U)) & ((1u << U) - 1);
    }
};

// The last of the 16 rows from `key` on that is in the plane.
__device__ __forceinline__ int last_row(const Params &p, int key) { return p.v.table ? 15 : min(15, p.v.R - 1 - key); }

// A row of a sequence with several chunks to D/4 lanes, which fold its partials in order.
template <int D, int ROWS>
__global__ __launch_bounds__(256) void merge_few_kernel(Params p) {
    constexpr int LPR = D / 4;
    const int of_seq = (blockIdx.x * 256 + threadIdx.x) / LPR, j = threadIdx.x % LPR, b = blockIdx.y;
    const int t = of_seq / p.Hq, hq = of_seq - t * p.Hq;
    if (t >= sequence(p, b).cnt) return;
    const int kvh = p.by_g(hq), r = t * p.G + hq - kvh * p.G;
    const int item = item_of(p, kvh, r / ROWS);
    const int2 chunk = p.chunks[static_cast<long long>(item) * p.v.B + b];   // written for the rows that exist
    if (chunk.y <= 1) return;                                // its one chunk wrote it
    const long long step = static_cast<long long>(p.v.H) * p.row_groups * ROWS;      // rows from chunk to chunk
    const long long first = chunk.x * step + static_cast<long long>(item) * ROWS + r % ROWS;
    float m = -INFINITY, l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    constexpr int U = 4;                                     // chunks in flight
    for (int s0 = 0; s0 < chunk.y; s0 += U) {
        float2 ml[U];
        float4 os[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (s0 + u >= chunk.y) break;
            ml[u] = *reinterpret_cast<const float2 *>(p.part_ml + (first + (s0 + u) * step) * 2);
            os[u] = *reinterpret_cast<const float4 *>(p.part_o + (first + (s0 + u) * step) * D + 4 * j);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (s0 + u >= chunk.y) break;
            fold(m, l, o, ml[u].x, ml[u].y, os[u]);
        }
    }
    const float f = l == 0.0f ? 0.0f : 1.0f / l;
    *reinterpret_cast<float4 *>(p.out + (static_cast<long long>(b) * p.T * p.Hq + of_seq) * D + 4 * j) =
        make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
}

// The merge of a call whose sequences have about p.quota / B chunks, and no more than there are positions for: from 16 on
// by a workgroup a row, which has all of them in flight. A sequence of 131072 keys in 64 chunks, 832 rows of 128: 9.0 us,
// by D/4 lanes a row 20.4 us; eight of 8192 keys in about 4, 16384 rows: 24.5 and 11.4 us.
template <int D, int ROWS>
void launch_merge(const Params &p, int least, hipStream_t s) {
    const long long chunks = std::min<long long>(p.quota / p.v.B, kv_capacity(p.v) / least);
    if (chunks >= 16) {
        hipLaunchKernelGGL((merge_kernel<Params, D, ROWS>), dim3(p.Hq, p.T, p.v.B), dim3(256), 0, s, p);
    } else {
        const long long lanes = static_cast<long long>(p.T) * p.Hq * (D / 4);
        hipLaunchKernelGGL((merge_few_kernel<D, ROWS>), dim3((lanes + 255) / 256, p.v.B), dim3(256), 0, s, p);
    }
}

// The rows kernel (kv_tree_rows.hip), p.row_groups blocks of kRowsBlock rows, and the merge.
void launch_rows(const Params &p, hipStream_t s);

}  // namespace kvt
}  // namespace aljabr
