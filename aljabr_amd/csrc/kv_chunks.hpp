// kv_chunks.hpp - work cut along the keys, for attention over caches whose
// lengths the host does not know: the cut of all sequences' keys into chunks
// of one size, and the merge of the chunks' partials. Shared by the attention
// over the 4-bit cache and over fp16 and fp32 caches (work_of and
// merge_rows_kernel are the 4-bit cache's alone).
//
// P, a kernel's parameters, has the cache's view v (sequences B, KV heads H),
// T, G, Hq, row_groups, quota, the dividers by_g, by_chunks (work_of: and by_items), the
// partials part_o, part_ml and chunks, and out; kEvenChunks: a sequence's
// chunks are of one size, instead of its last one taking what is left. Beside P
// stand
//   Seq sequence(const P &, int b)
//   bool row_tiles(const P &, const Seq &, int r0, int rows, int &a, int &z)
//   int item_of(const P &, int kvh, int group)
// The second gives the tiles [a, z) that rows [r0, r0 + rows) of a sequence see
// together; false when it has none of the rows. The third numbers KV heads and
// row groups for merge_kernel.
#pragma once

#include "device.hpp"

namespace aljabr {
namespace kv {

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

// A sequence's keys, its rows, and the position of the first of these.
struct Seq {
    int n, cnt, base;
};

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

// The size, a multiple of `least`, of `count` chunks of so many tiles. No more than the size that gave the count, so the
// last one is not empty.
__device__ __forceinline__ int even_size(int tiles, int count, int least) {
    const int each = (tiles + count - 1) / count;
    return (each + least - 1) / least * least;
}

// Chunk number w; b < 0 past the end. Called by whole waves.
template <class P>
__device__ __forceinline__ Chunk find_chunk(const P &p, int w, int r0, int rows, int least) {
    Chunk c{-1, 0, 0, 0, 0, 0, {0, 0, 0}};
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
        if constexpr (P::kEvenChunks) per = even_size(z - a, c.count, least);
        c.t0 = a + i * per;
        c.t1 = min(c.t0 + per, z);
        return c;
    }
    // A lane a sequence; the last (for B <= 64 the only) 64 stay in registers.
    const int last = (B - 1) & ~63;
    Seq s{0, 0, 0};
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
    float inv = __builtin_amdgcn_rcpf(static_cast<float>(per));
    // This lane's chunks, ceil((z - a) / per) and one for a sequence without keys: the estimate is at most one off.
    auto chunks = [&]() __attribute__((always_inline)) {
        int n = static_cast<int>(static_cast<float>(z - a) * inv);
        n += n * per < z - a ? 1 : 0;
        n -= n > 0 && (n - 1) * per >= z - a ? 1 : 0;
        n += n * per < z - a ? 1 : 0;
        return r0 < s.cnt * p.G ? max(n, 1) : 0;
    };
    if constexpr (P::kEvenChunks) {
        // What sequences take beyond the quota for their last chunks makes the chunks larger (up to 64 sequences, twice):
        // workgroups past what the chip holds at once would run alone.
        for (int i = 0; i < 2 && last == 0; ++i) {
            const int all = __builtin_amdgcn_readlane(wave_scan(chunks()), 63);
            if (all <= p.quota || B > p.quota) break;
            per = static_cast<int>(static_cast<float>(per) * static_cast<float>(all) * __builtin_amdgcn_rcpf(static_cast<float>(p.quota))) + 1;
            per = (per + least - 1) / least * least;
            inv = __builtin_amdgcn_rcpf(static_cast<float>(per));
        }
    }
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
        const int n = chunks();
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
            c.seq.base = __builtin_amdgcn_readlane(s.base, l);
            c.b = b0 + l;
            if constexpr (P::kEvenChunks) per = even_size(z - a, c.count, least);
            c.t0 = a + (w - c.first) * per;
            c.t1 = min(c.t0 + per, z);
            return c;
        }
        before = __builtin_amdgcn_readlane(end, 63);
        singles += __builtin_popcountll(single);
    }
    return c;
}

// The item and chunk number of a workgroup: `quota` chunks of every item, the
// chunk varying fastest, then the numbers that only uneven batches need (no CU
// is left half full by workgroups that find none).
template <class P>
__device__ __forceinline__ void work_of(const P &p, int id, int &item, int &w) {
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
template <class P, int D, int ROWS>
__global__ __launch_bounds__(256) void merge_kernel(P p) {
    constexpr int LPS = D / 4, SG = 256 / LPS;
    __shared__ float st[SG * (D + 2)];
    const int hq = blockIdx.x, t = blockIdx.y, b = blockIdx.z;
    const int kvh = p.by_g(hq), r = t * p.G + hq - kvh * p.G;
    const int item = item_of(p, kvh, r / ROWS);
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

// The row group of the item group i, and the other way round: the last, of most keys when causal, first.
template <class P>
__device__ __forceinline__ int group_of(const P &p, int i) { return p.row_groups - 1 - i; }

// A wave a row of a sequence with several chunks: D/4 lanes take a chunk's
// partial as float4s (64 / (D/4) chunks at once), folded in order, then across
// the lane groups.
template <class P, int D, int ROWS>
__global__ __launch_bounds__(256) void merge_rows_kernel(P p) {
    constexpr int LPS = D / 4, SG = 64 / LPS;
    const int of_seq = blockIdx.x * 4 + (threadIdx.x >> 6), b = blockIdx.y;
    const int t = of_seq / p.Hq, hq = of_seq - t * p.Hq;
    if (t >= p.T) return;
    const long long row = static_cast<long long>(b) * p.T * p.Hq + of_seq;
    const int kvh = p.by_g(hq), r = t * p.G + hq - kvh * p.G;
    const int item = group_of(p, r / ROWS) * p.v.H + kvh;
    const int2 chunk = p.chunks[static_cast<long long>(item) * p.v.B + b];   // written for the rows that exist
    if (t >= sequence(p, b).cnt || chunk.y <= 1) return;   // no row, or its one chunk wrote it
    const long long step = static_cast<long long>(p.v.H) * p.row_groups * ROWS;
    const long long first = chunk.x * step + static_cast<long long>(item) * ROWS + r % ROWS;
    const int lane = threadIdx.x & 63, sg = lane / LPS, j = lane % LPS;
    float m = -INFINITY, l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    constexpr int U = 4;                                   // chunks in flight per lane group
    for (int s0 = sg; s0 < chunk.y; s0 += U * SG) {
        float2 ml[U];
        float4 os[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long long s = s0 + u * SG < chunk.y ? s0 + u * SG : s0;
            ml[u] = *reinterpret_cast<const float2 *>(p.part_ml + (first + s * step) * 2);
            os[u] = *reinterpret_cast<const float4 *>(p.part_o + (first + s * step) * D + 4 * j);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (s0 + u * SG < chunk.y) fold(m, l, o, ml[u].x, ml[u].y, os[u]);
    }
#pragma unroll
    for (int off = LPS; off < 64; off <<= 1) {
        const float m2 = __shfl_xor(m, off), l2 = __shfl_xor(l, off);
        const float4 o2 = make_float4(__shfl_xor(o.x, off), __shfl_xor(o.y, off), __shfl_xor(o.z, off), __shfl_xor(o.w, off));
        fold(m, l, o, m2, l2, o2);
    }
    const float f = l == 0.0f ? 0.0f : 1.0f / l;
    if (sg == 0) *reinterpret_cast<float4 *>(p.out + row * D + 4 * j) = make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
}

}  // namespace kv
}  // namespace aljabr
