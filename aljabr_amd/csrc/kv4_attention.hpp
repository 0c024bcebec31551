// kv4_attention.hpp - what the two kernels of attention over the 4-bit cache
// share: the rows' key ranges and the decoder of codes. Included by the two
// .hip files only.
#pragma once

#include "device.hpp"
#include "internal.hpp"
#include "kv4.hpp"
#include "kv_chunks.hpp"

namespace aljabr {
namespace kv4 {

using namespace kv;

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

struct Params {
    static constexpr bool kEvenChunks = false;
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

__device__ __forceinline__ Seq sequence(const Params &p, int b) {
    Seq s;
    s.n = min(max(p.lens[b], 0), kv4_capacity(p.v));
    s.cnt = p.counts ? min(max(p.counts[b], 0), p.T) : p.T;
    s.base = s.n - s.cnt;
    return s;
}

__device__ __forceinline__ int item_of(const Params &p, int kvh, int group) { return kvh * p.row_groups + group; }

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

// The rows kernel (kv4_rows.hip), p.row_groups blocks of kRowsBlock rows, and the merge.
void launch_rows(const Params &p, hipStream_t s);

}  // namespace kv4
}  // namespace aljabr
