// kv4_attention.hpp - what the two kernels of attention over the 4-bit cache
// share: the rows' key ranges, the cut of the keys into chunks, the decoder of
// codes and the merge of chunks' partials. Included by the two .hip files only.
#pragma once

#include "device.hpp"
#include "internal.hpp"
#include "kv4.hpp"

namespace aljabr {
namespace kv4 {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 32;                    // keys a wave takes at once
// Waves of a workgroup, and tiles it takes at the least (two at D = 256, whose ring of tiles is twice as large).
__host__ __device__ constexpr int waves(int D) { return D == 256 ? 2 : 4; }
constexpr int kRowsBlock = 128;              // rows a workgroup of the rows kernel stacks
constexpr int kRowsLeast = 4;                // tiles it takes at the least
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kWeightScale = 8192.0f;      // weights are at most 4

// n / d for 0 <= n < 2^31 without a division.
struct FastDiv {
    uint32_t mul, shift;
    void set(uint32_t d) {
        uint32_t l = 0;
        while ((uint64_t{1} << l) < d) ++l;
        shift = 31 + l;
        mul = static_cast<uint32_t>(((uint64_t{1} << shift) + d - 1) / d);   // off by less than 1: n / 2^shift of it is below 1 / d
    }
    __device__ __forceinline__ int operator()(int n) const {
        return static_cast<int>(static_cast<uint64_t>(static_cast<uint32_t>(n)) * mul >> shift);
    }
};

struct Params {
    Kv4View v;
    float *out;
    const float *q;
    const int *lens, *counts;
    int T, Hq, G, row_groups;
    FastDiv by_g, by_groups, by_rows, by_chunks, by_items, by_heads;   // G, row_groups, rows of a block, chunks that vary fastest, H * row_groups, H
    float scale, unscale;                    // their product is the call's scale times log2(e)
    float soft_cap;
    int causal, window;
    int quota;                               // chunks that the keys of all sequences are cut into (about), 0: one each
    float *part_o, *part_ml;                 // per slot, KV head, row group and stacked row: D sums, and (m, l)
    int2 *chunks;                            // per sequence, KV head and row group: its first slot and its chunks
};

// A sequence's keys and its rows.
struct Seq {
    int n, cnt;
};
__device__ __forceinline__ Seq sequence(const Params &p, int b) {
    Seq s;
    s.n = min(max(p.lens[b], 0), kv4_capacity(p.v));
    s.cnt = p.counts ? min(max(p.counts[b], 0), p.T) : p.T;
    return s;
}

// Keys [lo, hi) that row t sees.
__device__ __forceinline__ void key_range(const Params &p, const Seq &s, int t, int &lo, int &hi) {
    const int pos = s.n - s.cnt + t;
    hi = p.causal ? max(pos + 1, 0) : s.n;
    lo = p.window > 0 ? max(pos - p.window + 1, 0) : 0;
}

// The tiles [a, z) that rows [r0, r0 + rows) of a sequence see together; false when it has none of the rows.
__device__ __forceinline__ bool row_tiles(const Params &p, const Seq &s, int r0, int rows, int &a, int &z) {
    a = z = 0;
    if (r0 >= s.cnt * p.G) return false;
    int lo, hi, x;
    key_range(p, s, p.by_g(r0), lo, x);
    key_range(p, s, min(p.by_g(r0 + rows - 1), s.cnt - 1), x, hi);
    a = lo / kTile;
    z = hi > lo ? (hi + kTile - 1) / kTile : a;
    return true;
}

// Inclusive sum over the lanes up to this one.
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);      // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);      // row 0's and 2's sums into 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);      // the first half's into the second
    return v;
}

// One chunk of the work of a row group: tiles [t0, t1) of sequence b. The
// tiles of all sequences are cut into chunks of one size, a multiple of
// `least`, about `quota` of them: a batch of uneven lengths keeps every
// workgroup busy alike. Chunks are numbered through the sequences, and slots
// of partials through those of several chunks (a single chunk writes its rows
// itself): fewer than 2 quota, as each of these is longer than one chunk, and
// fewer than quota + B (partial_slots).
struct Chunk {
    int b, t0, t1;
    int first, count;        // of the sequence's chunks
    int slot;                // of the first
    Seq seq;
};

// Chunk number w; b < 0 past the end. Called by whole waves.
__device__ __forceinline__ Chunk find_chunk(const Params &p, int w, int r0, int rows, int least) {
    Chunk c{-1, 0, 0, 0, 0, 0, {0, 0}};
    const int lane = threadIdx.x & 63, B = p.v.B;
    if (p.quota == 0 || B == 1) {
        const int b = p.quota ? 0 : w;
        int a, z;
        c.seq = sequence(p, b);
        if (!row_tiles(p, c.seq, r0, rows, a, z)) return c;
        int per = max(z - a, 1);
        if (p.quota) {
            per = max(p.by_chunks(z - a + p.quota - 1), least);
            per = (per + least - 1) / least * least;
            c.count = max((z - a + per - 1) / per, 1);
        } else {
            c.count = 1;
        }
        const int i = p.quota ? w : 0;
        if (i >= c.count) return c;
        c.b = b;
        c.first = p.quota ? 0 : b;
        c.t0 = a + i * per;
        c.t1 = min(c.t0 + per, z);
        return c;
    }
    // A lane a sequence; the last (for B <= 64 the only) 64 stay in registers.
    const int last = (B - 1) & ~63;
    Seq s{0, 0};
    int a = 0, z = 0, total = 0;
    for (int b0 = 0; b0 <= last; b0 += 64) {
        a = z = 0;
        if (b0 + lane < B) {
            s = sequence(p, b0 + lane);
            row_tiles(p, s, r0, rows, a, z);
        }
        total += __builtin_amdgcn_readlane(wave_scan(z - a), 63);
    }
    int per = max(p.by_chunks(total + p.quota - 1), least);
    per = (per + least - 1) / least * least;
    const float inv = __builtin_amdgcn_rcpf(static_cast<float>(per));
    int before = 0, singles = 0;                           // chunks, and sequences of one, of the groups of 64 before
    for (int b0 = 0; b0 <= last; b0 += 64) {
        if (last) {
            a = z = 0;
            s.cnt = 0;
            if (b0 + lane < B) {
                s = sequence(p, b0 + lane);
                row_tiles(p, s, r0, rows, a, z);
            }
        }
        // ceil((z - a) / per): the estimate is at most one off.
        int n = static_cast<int>(static_cast<float>(z - a) * inv);
        n += n * per < z - a ? 1 : 0;
        n -= n > 0 && (n - 1) * per >= z - a ? 1 : 0;
        n += n * per < z - a ? 1 : 0;
        n = r0 < s.cnt * p.G ? max(n, 1) : 0;
        const int end = before + wave_scan(n);
        const uint64_t single = __ballot(n == 1);
        const uint64_t hit = __ballot(w >= end - n && w < end);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            c.count = __builtin_amdgcn_readlane(n, l);
            c.first = __builtin_amdgcn_readlane(end, l) - c.count;
            c.slot = c.first - singles - __builtin_popcountll(single & ((uint64_t{1} << l) - 1));   // of one chunk: not used
            a = __builtin_amdgcn_readlane(a, l);
            z = __builtin_amdgcn_readlane(z, l);
            c.seq.n = __builtin_amdgcn_readlane(s.n, l);
            c.seq.cnt = __builtin_amdgcn_readlane(s.cnt, l);
            c.b = b0 + l;
            c.t0 = a + (w - c.first) * per;
            c.t1 = min(c.t0 + per, z);
            return c;
        }
        before = __builtin_amdgcn_readlane(end, 63);
        singles += __builtin_popcountll(single);
    }
    return c;
}

__device__ __forceinline__ half2v as_half2(uint32_t u) { return __builtin_bit_cast(half2v, u); }
__device__ __forceinline__ uint32_t as_u32(half2v h) { return __builtin_bit_cast(uint32_t, h); }
__device__ __forceinline__ half2v pair(float a, float b) {
    return half2v{static_cast<_Float16>(a), static_cast<_Float16>(b)};
}

// Masks in scalar and exponents in vector registers: one v_and_or_b32 each.
struct Magic {
    uint32_t m0 = 0x000f000fu, m4 = 0x00f000f0u, e10 = 0x64006400u, e6 = 0x54005400u;
    __device__ __forceinline__ Magic() { asm("" : "+s"(m0), "+s"(m4), "+v"(e10), "+v"(e6)); }
};

// The 8 nibbles of the 16-bit halves of w, in pairs (nibble i of the low half,
// nibble i of the high half), times the pair of scales d.
__device__ __forceinline__ void decode8(const Magic &g, uint32_t w, half2v d, uint32_t (&r)[4]) {
    const half2v o10 = {static_cast<_Float16>(-1032.0f), static_cast<_Float16>(-1032.0f)};
    const half2v o6 = {static_cast<_Float16>(-72.0f), static_cast<_Float16>(-72.0f)};
    const uint32_t x = w >> 8;
    r[0] = as_u32((as_half2((w & g.m0) | g.e10) + o10) * d);
    r[1] = as_u32((as_half2((w & g.m4) | g.e6) + o6) * d);
    r[2] = as_u32((as_half2((x & g.m0) | g.e10) + o10) * d);
    r[3] = as_u32((as_half2((x & g.m4) | g.e6) + o6) * d);
}

__device__ __forceinline__ half8 frag(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_bit_cast(half8, make_uint4(a, b, c, d));
}

__device__ __forceinline__ uint32_t lds_address(const void *p) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) void *)p));
}

// A scale that is not finite, or past the writer's largest (8160): a code times it may leave fp16.
__device__ __forceinline__ bool may_overflow(_Float16 x) {
    return (__builtin_bit_cast(uint16_t, x) & 0x7fffu) > 0x6ff8u;
}

// Whether one of the 8 values of w's nibbles is not a finite fp16 number.
__device__ __forceinline__ bool overflows(const Magic &g, uint32_t w, _Float16 d) {
    uint32_t f[4], all_ones = 0;
    decode8(g, w, half2v{d, d}, f);
#pragma unroll
    for (int i = 0; i < 4; ++i) all_ones |= (f[i] & 0x7fff7fffu) + 0x04000400u;      // the exponent's carry
    return all_ones & 0x80008000u;
}

// x of the lane 8 columns away (the row's other fp16 part).
__device__ __forceinline__ float other_part(float x) { return dpp_f32<0x128>(x); }

// Where a tile's two 16-key halves are (uniform over the wave).
struct Place {
    long long row[2];            // first key's row in the codes planes
    long long scale[2];          // and in the scales planes
    bool ok[2];                  // the half's block exists
};

template <int D, bool PAGED>
__device__ __forceinline__ Place place(const Params &p, int b, int kvh, int n_keys, int kt) {
    Place x;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        int key = kt * kTile + 16 * u;
        if (key >= n_keys) key = kt * kTile;               // past the end: the tile's first half again, masked
        int s = b, row = key;
        x.ok[u] = true;
        if constexpr (PAGED) {
            const int blk = p.by_rows(key);
            // A scalar load: nothing writes the table while the kernel runs.
            s = ((const __attribute__((address_space(4))) int *)p.v.table)[static_cast<long long>(b) * p.v.max_blocks + blk];
            row = key - blk * p.v.R;
            x.ok[u] = s >= 0 && s < p.v.num_blocks;
            if (!x.ok[u]) s = 0;
        }
        const long long head = static_cast<long long>(s) * p.v.H + kvh;
        x.row[u] = head * p.v.R + row;
        x.scale[u] = head * (D / 32) * p.v.R + row;
    }
    return x;
}

// The item and chunk number of a workgroup: `quota` chunks of every item, the
// chunk varying fastest, then the numbers that only uneven batches need (no CU
// is left half full by workgroups that find none).
__device__ __forceinline__ void work_of(const Params &p, int id, int &item, int &w) {
    const int most = p.quota ? p.quota : p.v.B, items = p.v.H * p.row_groups;
    item = p.by_chunks(id);
    w = id - item * most;
    if (item >= items) {
        w = most + p.by_items(id - items * most);
        item = id - w * items;
    }
}

// Folds the state (m2, l2, o2) into (m, l, o); a state without keys has m = -inf.
__device__ __forceinline__ void fold(float &m, float &l, float4 &o, float m2, float l2, const float4 &o2) {
    const float mn = fmaxf(m, m2);
    if (mn == -INFINITY) return;
    const float a = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
    const float e = m2 == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m2 - mn);
    l = fmaf(l, a, l2 * e);
    o.x = fmaf(o.x, a, o2.x * e);
    o.y = fmaf(o.y, a, o2.y * e);
    o.z = fmaf(o.z, a, o2.z * e);
    o.w = fmaf(o.w, a, o2.w * e);
    m = mn;
}

// One workgroup a row of a sequence with several chunks: D/4 lanes take a
// chunk's partial as float4s, 256 / (D/4) chunks at once, folded in order and
// then across the lane groups.
template <int D, int ROWS>
__global__ __launch_bounds__(256) void kv4_merge_kernel(Params p) {
    constexpr int LPS = D / 4, SG = 256 / LPS;
    __shared__ float st[SG * (D + 2)];
    const int hq = blockIdx.x, t = blockIdx.y, b = blockIdx.z;
    const int kvh = p.by_g(hq), r = t * p.G + hq - kvh * p.G;
    const int item = kvh * p.row_groups + r / ROWS;
    const int2 chunk = p.chunks[static_cast<long long>(item) * p.v.B + b];   // written for the rows that exist
    if (t >= sequence(p, b).cnt || chunk.y <= 1) return;   // no row, or its one chunk wrote it
    const int used = chunk.y;
    const long long row = (static_cast<long long>(b) * p.T + t) * p.Hq + hq;
    const long long step = static_cast<long long>(p.v.H) * p.row_groups * ROWS;      // rows from chunk to chunk
    const long long first = chunk.x * step + static_cast<long long>(item) * ROWS + r % ROWS;
    const float *po = p.part_o + first * D, *pm = p.part_ml + first * 2;
    const int sg = threadIdx.x / LPS, j = threadIdx.x % LPS;
    float m = -INFINITY, l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    constexpr int U = 8;                                   // splits in flight per lane group
    for (int s0 = sg; s0 < used; s0 += U * SG) {
        float ms[U], ls[U];
        float4 os[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long long s = s0 + u * SG < used ? s0 + u * SG : s0;
            const float2 ml = *reinterpret_cast<const float2 *>(pm + 2 * s * step);
            ms[u] = ml.x;
            ls[u] = ml.y;
            os[u] = *reinterpret_cast<const float4 *>(po + s * step * D + 4 * j);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (s0 + u * SG >= used) break;
            fold(m, l, o, ms[u], ls[u], os[u]);
        }
    }
    float *my = st + sg * (D + 2);
    my[4 * j] = o.x;
    my[4 * j + 1] = o.y;
    my[4 * j + 2] = o.z;
    my[4 * j + 3] = o.w;
    if (j == 0) {
        my[D] = m;
        my[D + 1] = l;
    }
    __syncthreads();
    for (int dd = threadIdx.x; dd < D; dd += 256) {
        float M = -INFINITY, L = 0.0f, O = 0.0f;
#pragma unroll
        for (int g = 0; g < SG; ++g) M = fmaxf(M, st[g * (D + 2) + D]);
        if (M != -INFINITY) {
#pragma unroll
            for (int g = 0; g < SG; ++g) {
                const float mg = st[g * (D + 2) + D];
                if (mg == -INFINITY) continue;
                const float e = __builtin_amdgcn_exp2f(mg - M);
                L = fmaf(st[g * (D + 2) + D + 1], e, L);
                O = fmaf(st[g * (D + 2) + dd], e, O);
            }
        }
        p.out[row * D + dd] = L == 0.0f ? 0.0f : O / L;
    }
}

// The rows kernel (kv4_rows.hip), p.row_groups blocks of kRowsBlock rows, and the merge.
void launch_rows(const Params &p, hipStream_t s);

}  // namespace kv4
}  // namespace aljabr
